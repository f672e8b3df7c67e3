"""Plain 64-bit restatements of the operators over a paged cache and on logits, and the rounding they are held to."""

import math
from collections import Counter

import torch

STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # half a step, relative


def make_cache(lengths, *, kv_heads, head_dim, page, dtype, slots_first=False, columns=None, extra=3, seed=0, spare=0):
    """Pools whose slots behind every sequence's end hold NaN and infinities, and tables with nonsense behind the last page.
    ``spare`` more slots per sequence are mapped (for tokens to come)."""
    generator = torch.Generator().manual_seed(seed)
    counts = [max(0, -(-(n + spare) // page)) if n >= 0 else 0 for n in lengths]
    total = sum(counts) + extra
    columns = columns or max([*counts, 1])
    order = torch.randperm(total, generator=generator).tolist()
    tables = torch.tensor([(-1, 1 << 30, -(1 << 31))[i % 3] for i in range(len(lengths) * columns)], dtype=torch.int32).view(len(lengths), columns)
    shape = (total, page, kv_heads, head_dim) if slots_first else (total, kv_heads, page, head_dim)
    keys, values = (torch.randn(shape, generator=generator) for _ in range(2))
    if slots_first:
        keys, values = keys.permute(0, 2, 1, 3), values.permute(0, 2, 1, 3)
    used = torch.zeros(total, page, dtype=torch.bool)
    for row, (n, count) in enumerate(zip(lengths, counts)):
        for column in range(count):
            tables[row, column] = order.pop()
            used[tables[row, column], :max(0, min(page, n - column * page))] = True
    wild = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(total * page) % 3].view(total, 1, page, 1)
    keys, values = (torch.where(used[:, None, :, None], data, wild).to(dtype) for data in (keys, values))
    weights = torch.rand(total, kv_heads, page, generator=generator) * 3
    if slots_first:      # torch.where made them contiguous: the slots of a page lie first again
        keys, values = (data.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for data in (keys, values))
    return keys, values, tables, weights


def slots_of(pool, table, length):
    """The first ``length`` slots of a sequence, [heads, length, ...]."""
    page = pool.shape[2]
    return pool[table[:-(-length // page)].long()].transpose(0, 1).flatten(1, 2)[:, :length]


def rotated(x, position, theta):
    """Rotate-half pairing of [heads, width] by ``position``, in 64 bits."""
    half = x.shape[-1] // 2
    angle = position * theta ** (-torch.arange(half, dtype=torch.float64) / half)
    low, high = x[..., :half].double(), x[..., half:].double()
    return torch.cat((low * angle.cos() - high * angle.sin(), high * angle.cos() + low * angle.sin()), -1)


def attend(q, keys, values, scale, dtype, rotary):
    """``(out, bound, share, slack)`` of one sequence: q [q_heads, width] in 64 bits, keys and values [kv_heads, n, width].

    ``slack`` bounds the error of a score, hence the relative error of exp(score): products of 16-bit values are exact in
    fp32 and a dot product of D of them is off by at most D + 4 steps of 2^-23 (truncating adders) of sum |q k|; a rotated
    query is held in two 16-bit parts, 2^-17 of it at most left out.  exp2 and the division add some steps of 2^-22.  The output
    adds the rounding of the softmax weights to the cache's type (``step`` of sum w |v|) and its own (``step`` of |out|)."""
    heads, n, width = keys.shape
    grouped = q.view(heads, -1, width)
    scores = torch.einsum("hgd,hpd->hgp", grouped, keys.double()) * scale
    share = torch.softmax(scores, -1)
    size = (torch.einsum("hgd,hpd->hgp", grouped.abs(), keys.double().abs()) * abs(scale)).amax(-1, keepdim=True)
    slack = size * ((width + 4) * 2.0 ** -23 + (2.0 ** -17 if rotary else 0)) * 2 + 2.0 ** -20
    out = torch.einsum("hgp,hpd->hgd", share, values.double())
    mass = torch.einsum("hgp,hpd->hgd", share, values.double().abs())
    bound = STEP[dtype] * (out.abs() + mass) + slack * mass + 2.0 ** -25   # the last: fp16 outputs below its normal range
    return out.reshape(-1, width), bound.reshape(-1, width), share, slack


def evicted(weight, budget, sinks, recent):
    """Kept slots of one head, ascending: ``weight`` [n]."""
    n = weight.numel()
    if n <= budget:
        return list(range(n))
    safe = [p for p in range(n) if p < sinks or p >= n - recent]
    rank = lambda p: (-math.inf if math.isnan(float(weight[p])) else float(weight[p]))
    middle = sorted((p for p in range(n) if sinks <= p < n - recent),
                    key=lambda p: (math.isnan(float(weight[p])), -rank(p), p))
    return sorted(safe + middle[:budget - len(safe)])


def adjusted(row, offset, *, history=(), prompt=0, repetition=1.0, frequency=0.0, presence=0.0, biases=(), mask=None):
    """One row of logits in 64 bits."""
    x = row.double().clone()
    generated = Counter(history[max(prompt, 0):])
    for token in set(history):
        i = token - offset
        if not 0 <= i < x.numel():
            continue
        x[i] = x[i] / repetition if x[i] > 0 else x[i] * repetition
        count = generated[token]
        x[i] -= frequency * count + (presence if count else 0.0)
    for token, value in biases:
        if 0 <= token - offset < x.numel():
            x[token - offset] += value
    if mask is not None:
        for i in range(x.numel()):
            token = offset + i
            if not (int(mask[token // 32]) >> (token % 32)) & 1:
                x[i] = -math.inf
    return x
