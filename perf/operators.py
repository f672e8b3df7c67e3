"""Operators of a serving step over a paged cache, as cases to prepare, run, count and check.

Three operators, which a decode step calls one after another:

* ``attention``: one new token of every sequence attends to its paged key-value cache.  With ``rope`` the call takes the
  projected q | k | v, rotates q and k, stores k and v in the cache and attends; without it takes rotated queries and only
  reads.  With ``weights`` it also adds each slot's attention weight to an accumulator that lies in pages of its own.
* ``evict``: the heaviest slots of every sequence by that accumulator, its first and its latest ones, move to fresh pages.
* ``logits``: penalties for repeated tokens, sparse biases and a grammar's bit mask on the logits, and the greedy pick.

``run`` computes them in elementary torch operations, or, with ``own``, calls the framework.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA = 500000.0


def attention(name, rows, q_heads, kv_heads, head_dim, page, shortest, longest, dtype, rope, weights, slots_first=False):
    return {"name": name, "op": "attention", "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "shortest": shortest, "longest": longest, "dtype": dtype, "rope": rope, "weights": weights,
            "slots_first": slots_first}


def evict(name, rows, kv_heads, head_dim, page, shortest, longest, budget, sinks, recent, dtype, slots_first=False):
    return {"name": name, "op": "evict", "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "shortest": shortest, "longest": longest, "budget": budget, "sinks": sinks, "recent": recent, "dtype": dtype,
            "slots_first": slots_first}


def logits(name, rows, vocab, first, shard, history, biases, mask, dtype):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "first": first, "shard": shard, "history": history,
            "biases": biases, "mask": mask, "dtype": dtype}


def listed():
    return [
        # one conversation at its beginning, 8B-sized heads: a call that is all latency
        attention("attend one short", 1, 32, 8, 128, 16, 300, 300, "fp16", True, False),
        # the decoder's usual batch and context
        attention("attend eight of 1k", 8, 32, 8, 128, 16, 1024, 1024, "fp16", True, False),
        # one of eight ranks of the 70B-sized model: one key-value head, ragged long contexts, weights kept for eviction
        attention("attend a rank's shard", 8, 8, 1, 128, 64, 2000, 30000, "fp16", True, True),
        # one document of 128k tokens, all heads on one device, pages laid out slot by slot
        attention("attend one of 128k", 1, 64, 8, 128, 64, 131071, 131071, "bf16", False, False, True),
        # a full serving batch with contexts from some hundred tokens to 16k: the largest
        attention("attend a ragged batch", 64, 32, 8, 128, 16, 500, 16384, "bf16", True, False),
        # ungrouped heads of 64, odd lengths and pages, weights kept
        attention("attend ungrouped heads", 12, 14, 14, 64, 24, 17, 3001, "bf16", False, True),
        # a sequence that ran over its budget by some pages
        evict("evict a little", 1, 8, 128, 16, 2304, 2304, 2048, 4, 256, "fp16"),
        # a batch of long prompts cut to what the budget holds
        evict("evict long prompts", 16, 8, 128, 16, 5000, 16384, 4096, 4, 512, "bf16"),
        # one conversation's logits, a short history, no mask
        logits("penalties of one row", 1, 128256, 0, 128256, 300, 0, False, "fp16"),
        # a rank's vocabulary shard for the decoder's usual batch
        logits("penalties of a shard", 8, 128256, 16032, 16032, 1500, 20, True, "fp16"),
        # a serving batch with long histories, biases and grammars
        logits("penalties of a batch", 128, 128256, 0, 128256, 4000, 300, True, "bf16"),
        # the same in 32 bits at an odd vocabulary
        logits("penalties in 32 bits", 17, 50257, 0, 50257, 900, 7, True, "fp32"),
    ]


def log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "evict", "logits"))
    if kind == "logits":
        vocab = log_between(rng, 1000, 160000)
        first = rng.choice((0, 0, vocab // 2 + rng.randrange(40)))
        rows = min(log_between(rng, 1, 128), max(1, (1 << 24) // vocab))
        return logits("", rows, vocab, first, vocab - first, log_between(rng, 1, 6000), rng.choice((0, 1, 40, 300)),
                      rng.random() < 0.6, rng.choice(("fp16", "bf16", "fp32")))
    head_dim, page = rng.choice((64, 128, 128, 192, 256)), rng.choice((1, 8, 16, 16, 24, 32, 64, 100, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 10))
    longest = log_between(rng, 2, 30000)
    shortest = max(1, longest // rng.choice((1, 1, 3, 40)))
    rows = min(log_between(rng, 1, 64), max(1, (1 << (27 if kind == "attention" else 26)) // (longest * kv_heads * head_dim)))
    dtype, slots_first = rng.choice(("fp16", "bf16")), rng.random() < 0.5
    if kind == "attention":
        return attention("", rows, kv_heads * rng.choice((1, 2, 4, 4, 5, 8, 8, 12, 16)), kv_heads, head_dim, page, shortest,
                         longest, dtype, rng.random() < 0.5, rng.random() < 0.35, slots_first)
    budget = max(2, int(longest * rng.uniform(0.2, 1.1)))
    sinks = rng.choice((0, min(4, budget // 2)))
    return evict("", rows, kv_heads, head_dim, page, shortest, longest, budget, sinks, int((budget - sinks) * rng.choice((0, 0.1, 0.5))),
                 dtype, slots_first)


# ------------------------------------------------------------------------------------------------ inputs


def lengths_of(case):
    """Tokens held by each sequence, spread evenly over the logarithm; the last row of eight or more is a padded one."""
    rows, low, high = case["rows"], case["shortest"], case["longest"]
    spread = [int(round(high * (low / high) ** (i / max(1, rows - 1)))) for i in range(rows)]
    if rows >= 8:
        spread[-1] = -1
    return spread


def pool(case, pages, generator):
    """Keys or values in pages: [pages, heads, slots, head_dim], as the heads or the slots of a page lie first."""
    heads, page, width = case["kv_heads"], case["page"], case["head_dim"]
    shape = (pages, page, heads, width) if case["slots_first"] else (pages, heads, page, width)
    data = torch.randn(shape, device="cuda", dtype=DTYPES[case["dtype"]], generator=generator)
    return data.permute(0, 2, 1, 3) if case["slots_first"] else data


def page_tables(counts, order, columns):
    """Page ids of every row, -1 behind its last page; rows take their pages from ``order`` one after another."""
    starts = torch.cumsum(counts, 0) - counts
    column = torch.arange(columns, device="cuda")
    at = (starts[:, None] + column).clamp(max=order.numel() - 1)
    return torch.where(column < counts[:, None], order[at], -1).to(torch.int32)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    random = lambda *shape: torch.rand(shape, device="cuda", generator=generator)
    if case["op"] == "logits":
        return prepare_logits(case, generator, random)
    rows, page, heads, width = case["rows"], case["page"], case["kv_heads"], case["head_dim"]
    dtype = DTYPES[case["dtype"]]
    shuffle = torch.randperm(rows, device="cuda", generator=generator)
    lengths = torch.tensor(lengths_of(case), device="cuda")[shuffle]
    more = 1 if case["op"] == "attention" and case["rope"] else 0
    counts = (lengths.clamp(min=-1) + more + page - 1).clamp(min=0) // page
    budget = case.get("budget", 0)
    fresh = (lengths.clamp(min=0, max=budget) + page - 1) // page
    total = int(counts.sum() + fresh.sum()) + 3
    order = torch.randperm(total, device="cuda", generator=generator)
    state = {
        "case": case, "lengths": lengths.to(torch.int32),
        "tables": page_tables(counts, order, max(1, -(-(case["longest"] + more) // page))),
        "k_pages": pool(case, total, generator), "v_pages": pool(case, total, generator),
    }
    if case["op"] == "evict":
        left = order[int(counts.sum()):]
        state["new_tables"] = page_tables(fresh, left, max(1, -(-budget // page)))
        # most slots are hardly looked at and have the same small weight, few are looked at often
        drawn = random(total, heads, page)
        state["weights"] = torch.where(drawn < 0.3, 0.0078125, (-torch.log(drawn)) ** 3 * 4)
        return state
    state["out"] = torch.empty(rows, case["q_heads"], width, device="cuda", dtype=dtype)
    state["weights"] = (-torch.log(random(total, heads, page).clamp(min=1e-6))) ** 3 if case["weights"] else None
    if case["rope"]:
        state["qkv"] = torch.randn(rows, (case["q_heads"] + 2 * heads) * width, device="cuda", dtype=dtype, generator=generator)
        # a sequence whose cache was evicted from before is further on than its cache is long
        state["positions"] = (lengths.clamp(min=0) + torch.randint(0, 300, (rows,), device="cuda", generator=generator)).to(torch.int32)
    else:
        state["q"] = torch.randn(rows, case["q_heads"], width, device="cuda", dtype=dtype, generator=generator)
    return state


def prepare_logits(case, generator, random):
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    state = {"case": case, "out": torch.empty(rows, case["shard"], device="cuda", dtype=dtype),
             "picked": torch.empty(rows, device="cuda", dtype=torch.int64)}
    state["logits"] = (torch.randn(rows, case["shard"], device="cuda", generator=generator) * 3).to(dtype)
    # texts repeat themselves: token ids are drawn towards the low end
    state["tokens"] = (random(rows, case["history"]) ** 4 * vocab).to(torch.int64).clamp(max=vocab - 1)
    state["lengths"] = (random(rows) * (case["history"] // 2 + 1) + case["history"] - case["history"] // 2).to(torch.int32).clamp(max=case["history"])
    state["prompts"] = (state["lengths"] * random(rows)).to(torch.int32)
    state["repetition"] = 1.0 + random(rows) * 0.4
    state["frequency"], state["presence"] = random(rows) * 0.5, random(rows)
    state["bias_tokens"] = state["bias"] = state["mask"] = None
    if case["biases"]:
        state["bias_tokens"] = torch.randint(-1, vocab, (rows, case["biases"]), device="cuda", dtype=torch.int32, generator=generator)
        state["bias"] = torch.randn(rows, case["biases"], device="cuda", generator=generator) * 4
    if case["mask"]:
        words = torch.randint(-(1 << 31), 1 << 31, (rows, -(-vocab // 32)), device="cuda", generator=generator)
        # a grammar allows few tokens in most places
        state["mask"] = (words & words.roll(1, 1) & words.roll(3, 1)).to(torch.int32)
    return state


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return run_attention(state)
    return run_evict(state) if op == "evict" else run_logits(state)


def run_attention(state):
    case = state["case"]
    if own:
        from mlkit_b200 import kernels
        if case["rope"]:
            kernels.paged_rope_attention_decode(
                state["qkv"], state["positions"], state["lengths"], state["k_pages"], state["v_pages"], state["tables"],
                state["out"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"], theta=THETA,
                weights=state["weights"])
        else:
            kernels.paged_attention_decode(state["q"], state["lengths"], state["k_pages"], state["v_pages"], state["tables"],
                                           state["out"], weights=state["weights"])
        return attention_outputs(state, state["out"])
    lengths = state["lengths"].long()
    if case["rope"]:
        q, lengths = append(state)
    else:
        q = state["q"].float()
    rows, kv_heads, width, page = case["rows"], case["kv_heads"], case["head_dim"], case["page"]
    slot = torch.arange(state["tables"].shape[1] * page, device="cuda")
    held = slot < lengths[:, None]                                                        # [rows, slots]
    pages = state["tables"].long().clamp(min=0)[:, slot // page]
    keep = held[:, None, :, None]
    keys = torch.where(keep, state["k_pages"][pages, :, slot % page].permute(0, 2, 1, 3).float(), 0)
    scores = torch.matmul(q.view(rows, kv_heads, -1, width), keys.transpose(2, 3)) * width ** -0.5
    del keys
    scores = torch.where(held[:, None, None], scores, -math.inf)
    top = scores.amax(3, keepdim=True)
    weight = torch.exp(scores - torch.where(top > -math.inf, top, 0))
    weight = weight / weight.sum(3, keepdim=True).clamp(min=1e-38)
    values = torch.where(keep, state["v_pages"][pages, :, slot % page].permute(0, 2, 1, 3).float(), 0)
    out = torch.matmul(weight, values).view(rows, case["q_heads"], width).to(DTYPES[case["dtype"]])
    if case["weights"]:
        row, at = torch.nonzero(held, as_tuple=True)
        add, into = weight.sum(2)[row, :, at], (pages[row, at], slice(None), at % page)
        before = state["weights"][into]
        if case["rope"]:
            before = torch.where((at == lengths[row] - 1)[:, None], 0, before)            # the new slot begins at nothing
        state["weights"][into] = before + add
    return attention_outputs(state, out)


def attention_outputs(state, out):
    case, given = state["case"], {"out": out}
    if case["rope"]:
        given["k_pages"], given["v_pages"] = state["k_pages"], state["v_pages"]
    if case["weights"]:
        given["weights"] = state["weights"]
    return given


def append(state):
    """Rotates q and k of the projected rows and stores k and v behind each sequence; the queries and the new lengths."""
    case, lengths = state["case"], state["lengths"].long()
    rows, heads, width, page = case["rows"], case["kv_heads"], case["head_dim"], case["page"]
    half = width // 2
    q, k, v = state["qkv"].view(rows, -1, width).split((case["q_heads"], heads, heads), 1)
    turn = state["positions"].double()[:, None] * THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    cosine, sine = torch.cos(turn).float()[:, None], torch.sin(turn).float()[:, None]
    turned = lambda x: torch.cat((x[..., :half].float() * cosine - x[..., half:].float() * sine,
                                  x[..., half:].float() * cosine + x[..., :half].float() * sine), 2)
    row = torch.nonzero(lengths >= 0)[:, 0]
    at = lengths[row]
    pages = state["tables"].long()[row, at // page]
    state["k_pages"][pages, :, at % page] = turned(k)[row].to(state["k_pages"].dtype)
    state["v_pages"][pages, :, at % page] = v[row]
    return turned(q), torch.where(lengths >= 0, lengths + 1, 0)


def run_evict(state):
    case = state["case"]
    if own:
        from mlkit_b200 import kernels
        kept = kernels.evict_pages(state["k_pages"], state["v_pages"], state["weights"], state["tables"], state["lengths"],
                                   state["new_tables"], budget=case["budget"], sinks=case["sinks"], recent=case["recent"])
        return {"kept": kept, "keys": state["k_pages"], "values": state["v_pages"], "weights": state["weights"]}
    page, budget = case["page"], case["budget"]
    lengths = state["lengths"].long().clamp(min=0)[:, None]
    slot = torch.arange(max(budget, state["tables"].shape[1] * page), device="cuda")
    pages = state["tables"].long().clamp(min=0)[:, (slot // page).clamp(max=state["tables"].shape[1] - 1)]
    score = state["weights"][pages, :, slot % page].permute(0, 2, 1)                     # [rows, heads, slots]
    safe = (slot < case["sinks"]) | (slot >= lengths - case["recent"])
    score = torch.where(safe[:, None], math.inf, score)
    score = torch.where((slot < lengths)[:, None], score, -math.inf)
    best = torch.sort(score, dim=2, descending=True, stable=True)[1][:, :, :budget]
    best = torch.where(best < lengths[:, None], best, slot.numel())
    kept = torch.sort(best, dim=2)[0]
    kept = torch.where(kept < slot.numel(), kept, -1)
    row, head, new = torch.nonzero(kept >= 0, as_tuple=True)
    old = kept[row, head, new]
    source = (state["tables"].long()[row, old // page], head, old % page)
    target = (state["new_tables"].long()[row, new // page], head, new % page)
    state["k_pages"][target] = state["k_pages"][source]
    state["v_pages"][target] = state["v_pages"][source]
    state["weights"][target] = state["weights"][source]
    return {"kept": kept.to(torch.int32), "keys": state["k_pages"], "values": state["v_pages"], "weights": state["weights"]}


def run_logits(state):
    case = state["case"]
    if own:
        from mlkit_b200 import kernels
        kernels.adjust_logits(state["logits"], tokens=state["tokens"], lengths=state["lengths"], prompts=state["prompts"],
                              repetition=state["repetition"], frequency=state["frequency"], presence=state["presence"],
                              bias_tokens=state["bias_tokens"], bias=state["bias"], mask=state["mask"], offset=case["first"],
                              picked=state["picked"], out=state["out"])
        return {"logits": state["out"], "token": state["picked"]}
    rows, vocab, x = case["rows"], case["vocab"], state["logits"].float()
    column = slice(case["first"], case["first"] + case["shard"])
    at = torch.arange(case["history"], device="cuda")
    held = at < state["lengths"][:, None]
    zeros = torch.zeros(rows, vocab, device="cuda", dtype=torch.int32)
    seen = zeros.scatter_add(1, state["tokens"], held.int())[:, column] > 0
    count = zeros.scatter_add(1, state["tokens"], (held & (at >= state["prompts"][:, None])).int())[:, column]
    penalty = state["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / penalty, x * penalty), x)
    x = x - state["frequency"][:, None] * count
    x = x - torch.where(count > 0, state["presence"][:, None], 0)
    if case["biases"]:
        given = state["bias_tokens"].long()
        dense = torch.zeros(rows, vocab, device="cuda", dtype=torch.float64)
        dense.scatter_add_(1, given.clamp(min=0), torch.where(given >= 0, state["bias"], 0).double())
        x = x + dense[:, column].float()
    if case["mask"]:
        token = torch.arange(case["first"], case["first"] + case["shard"], device="cuda")
        allowed = (state["mask"][:, token // 32] >> (token % 32).int()) & 1
        x = torch.where(allowed > 0, x, -math.inf)
    x = x.to(state["logits"].dtype)
    return {"logits": x, "token": case["first"] + first_best(x)}


def first_best(x):
    """The lowest index of the largest value of each row."""
    index = torch.arange(x.shape[1], device="cuda")
    return torch.where(x == x.amax(1, keepdim=True), index, x.shape[1]).amin(1)


# ------------------------------------------------------------------------------------------------ counts


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    rows = case["rows"]
    if case["op"] == "logits":
        history = rows * case["history"] * 3 // 4
        moved = 2 * size * rows * case["shard"] + 8 * history + 8 * rows * case["biases"] + 8 * rows
        return {"bytes": moved + (rows * case["shard"] // 8 if case["mask"] else 0), "flops": rows * case["shard"]}
    row_bytes = case["head_dim"] * size
    held = [max(0, n) for n in lengths_of(case)]
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in held)
        return {"bytes": case["kv_heads"] * (4 * sum(held) + kept * (4 * row_bytes + 4 + 4)), "flops": 0}
    slots = sum(held) * case["kv_heads"]
    moved = 2 * slots * row_bytes + (8 * slots if case["weights"] else 0) + 2 * rows * case["q_heads"] * row_bytes
    if case["rope"]:
        moved += 4 * rows * case["kv_heads"] * row_bytes
    return {"bytes": moved, "flops": 4 * sum(held) * case["q_heads"] * case["head_dim"]}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": exact_attention, "evict": exact_evict, "logits": exact_logits}[case["op"]](case, state)


def rows_of_pages(pages, table, length, page):
    """One sequence's slots in order, [heads, length, ...]: its pages side by side, in 64 bits."""
    count = -(-length // page)
    joined = pages[table[:count].long()].double()
    return joined.transpose(0, 1).flatten(1, 2)[:, :length]


def exact_attention(case, state):
    groups, heads, width, page = case["q_heads"] // case["kv_heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(case["rows"], case["q_heads"], width, device="cuda", dtype=torch.float64)
    sums = state["weights"].double() if case["weights"] else None
    k_pages, v_pages = (state[name].double() if case["rope"] else state[name] for name in ("k_pages", "v_pages"))
    for m, length in enumerate(state["lengths"].tolist()):
        table = state["tables"][m]
        if length < 0:
            continue
        keys = rows_of_pages(k_pages, table, length, page)
        values = rows_of_pages(v_pages, table, length, page)
        if case["rope"]:
            parts = state["qkv"][m].double().view(-1, 2, width // 2)
            frequency = torch.pow(torch.tensor(THETA, device="cuda", dtype=torch.float64), -2 * torch.arange(width // 2, device="cuda").double() / width)
            turn = torch.polar(torch.ones_like(frequency), frequency * int(state["positions"][m]))
            turned = torch.complex(parts[:, 0], parts[:, 1]) * turn
            turned = torch.cat((turned.real, turned.imag), 1)
            query = turned[:case["q_heads"]]
            v_new = parts[case["q_heads"] + heads:].flatten(1)
            k_new = turned[case["q_heads"]:case["q_heads"] + heads].to(DTYPES[case["dtype"]]).double()  # as the cache holds it
            keys, values = torch.cat((keys, k_new[:, None]), 1), torch.cat((values, v_new[:, None]), 1)
            k_pages[table[length // page].long(), :, length % page] = k_new
            v_pages[table[length // page].long(), :, length % page] = v_new
        else:
            query = state["q"][m].double()
        if not keys.shape[1]:
            continue
        scores = torch.einsum("hgd,hpd->hgp", query.view(heads, groups, width), keys) / math.sqrt(width)
        share = torch.softmax(scores, 2)
        out[m] = torch.einsum("hgp,hpd->hgd", share, values).reshape(-1, width)
        if sums is not None:
            slot = torch.arange(keys.shape[1], device="cuda")
            into = (table[slot // page].long(), slice(None), slot % page)
            if case["rope"]:
                sums[table[length // page].long(), :, length % page] = 0
            sums[into] += share.sum(1).t()
    given = {"out": out}
    if case["rope"]:
        given["k_pages"], given["v_pages"] = k_pages, v_pages
    if sums is not None:
        given["weights"] = sums
    return given


def exact_evict(case, state):
    kept = torch.full((case["rows"], case["kv_heads"], case["budget"]), -1, device="cuda", dtype=torch.int32)
    pools = [state[name].double() for name in ("k_pages", "v_pages", "weights")]
    page = case["page"]
    for m, length in enumerate(state["lengths"].tolist()):
        take = min(case["budget"], length)
        if take <= 0:
            continue
        old, new = state["tables"][m].long(), state["new_tables"][m].long()
        weight = rows_of_pages(state["weights"], old, length, page)
        weight[:, :case["sinks"]] = weight[:, max(0, length - case["recent"]):] = math.inf
        for h in range(case["kv_heads"]):
            edge = torch.topk(weight[h], take)[0][-1]
            above, level = torch.nonzero(weight[h] > edge)[:, 0], torch.nonzero(weight[h] == edge)[:, 0]
            chosen = torch.cat((above, level[:take - above.numel()])).sort()[0]
            kept[m, h, :take] = chosen.to(torch.int32)
            to = torch.arange(take, device="cuda")
            for data in pools:
                data[new[to // page], h, to % page] = data[old[chosen // page], h, chosen % page]
    return {"kept": kept, "keys": pools[0], "values": pools[1], "weights": pools[2]}


def exact_logits(case, state):
    x = state["logits"].double()
    for m in range(case["rows"]):
        length, prompt = int(state["lengths"][m]), int(state["prompts"][m])
        history = state["tokens"][m, :length]
        total = torch.bincount(history, minlength=case["vocab"])
        count = torch.bincount(history[prompt:], minlength=case["vocab"])
        total, count = (c[case["first"]:case["first"] + case["shard"]].double() for c in (total, count))
        penalty = state["repetition"][m].double()
        row = torch.where(total > 0, torch.where(x[m] > 0, x[m] / penalty, x[m] * penalty), x[m])
        row = row - state["frequency"][m].double() * count - state["presence"][m].double() * count.clamp(max=1)
        if case["biases"]:
            entry, value = state["bias_tokens"][m].long(), state["bias"][m].double()
            inside = (entry >= case["first"]) & (entry < case["first"] + case["shard"])
            row = row.index_add(0, entry[inside] - case["first"], value[inside])
        if case["mask"]:
            bits = (state["mask"][m].long()[:, None] >> torch.arange(32, device="cuda")) & 1
            row = row.masked_fill(bits.flatten()[case["first"]:case["first"] + case["shard"]] == 0, -math.inf)
        x[m] = row
    return {"logits": x, "token": None}
