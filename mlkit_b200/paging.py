"""What a serving loop keeps between decode steps: ``PagedCache``, the keys and values of its sequences in pages, and
``LogitRules``, the penalties, biases and masks of its rows.

Neither has a counterpart in the reference, which leaves cache and sampling to ``transformers``
(``src/mlkit/inference/optimization.py:86-99`` compiles the model with its static cache).  ``TensorParallelDecoder`` takes
both; other callers use them with ``kernels.paged_rope_attention_decode``, ``kernels.evict_pages`` and
``kernels.adjust_logits``, which they hold the arguments of.
"""

from collections.abc import Iterable, Iterator, Mapping, Sequence
from contextlib import contextmanager

import torch
from torch import Tensor

from mlkit_b200 import kernels

HEAD_WIDTHS = (64, 128, 192, 256)


class PagedCache:
    """Keys and values of up to ``rows`` sequences for every layer, in pages of ``page`` slots taken from one pool per layer.

    All layers share the tables (``tables`` int32 [rows, columns]) and the lengths (``lengths`` int32 [rows], -1 for a row that
    is not in use); a page number means the same page of every layer's pool.  Pages are taken when a sequence needs
    them and given back when it ends, so the pool may be much smaller than ``rows * columns`` pages.  With ``track_weights`` every
    slot's attention weight is added up, and ``evict`` can cut sequences down to a budget of slots.

    The bookkeeping is on the host (``held`` mirrors ``lengths``): a step calls ``prepare`` before its launches and ``advance``
    after them.  On the device that is the addition to ``lengths`` and, when sequences begin pages, one copy of their numbers from
    pinned memory into ``tables``, so captured steps replay without synchronising; opening, releasing and evicting do not wait
    either.
    """

    def __init__(self, *, rows: int, columns: int, kv_heads: int, head_dim: int, page: int = 16, pages: int | None = None,
                 layers: int = 0, dtype: torch.dtype = torch.float16, device: torch.device | str = "cuda",
                 track_weights: bool = False) -> None:
        if rows < 1 or columns < 1 or page < 1 or kv_heads < 1 or layers < 0:
            raise ValueError("a paged cache needs rows, columns, heads and a page of at least one")
        if head_dim not in HEAD_WIDTHS:
            raise ValueError(f"a paged cache has heads of {HEAD_WIDTHS}, not of {head_dim}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a paged cache holds fp16 or bf16, not {dtype}")
        self.rows, self.columns, self.page, self.device = rows, columns, page, torch.device(device)
        self.pages = rows * columns if pages is None else pages
        if self.pages < 1:
            raise ValueError("a paged cache needs pages")
        self.shape, self.dtype, self.track_weights = (self.pages, kv_heads, page, head_dim), dtype, track_weights
        self.k_pages: list[Tensor] = []
        self.v_pages: list[Tensor] = []
        self.weights: list[Tensor] = []
        self.tables = torch.full((rows, columns), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.full((rows,), -1, dtype=torch.int32, device=self.device)
        self.held: list[int] = [-1] * rows
        self.owned: list[list[int]] = [[] for _ in range(rows)]
        self.free: list[int] = list(range(self.pages - 1, -1, -1))
        self._idle = False
        for _ in range(layers):
            self.add_layer()

    def add_layer(self) -> None:
        self.k_pages.append(torch.zeros(self.shape, dtype=self.dtype, device=self.device))
        self.v_pages.append(torch.zeros(self.shape, dtype=self.dtype, device=self.device))
        if self.track_weights:
            self.weights.append(torch.zeros(self.shape[:3], dtype=torch.float32, device=self.device))

    @property
    def capacity(self) -> int:
        """Slots a sequence can hold."""
        return self.columns * self.page

    # -- sequences --
    def open(self, row: int) -> None:
        """Begin a sequence in a row that is not in use."""
        if self.held[row] >= 0:
            raise ValueError(f"row {row} is in use")
        self.held[row] = 0
        self.lengths[row].fill_(0)

    def release(self, row: int) -> None:
        """End a row's sequence, if it has one, and give its pages back."""
        self.free.extend(reversed(self.owned[row]))
        self.owned[row], self.held[row] = [], -1
        self.lengths[row].fill_(-1)

    def reserve(self, row: int, slots: int) -> None:
        """Take the pages that ``slots`` slots of the row's sequence need, all of them or, with an error, none."""
        self._reserve([(row, slots)])

    def _reserve(self, wanted: Iterable[tuple[int, int]]) -> None:
        counts: list[tuple[int, int]] = []
        for row, slots in wanted:
            if self.held[row] < 0:
                raise ValueError(f"row {row} is not in use")
            if slots > self.capacity:
                raise ValueError(f"a sequence of {slots} slots exceeds the {self.columns} pages of {self.page} of a row")
            counts.append((row, max(0, -(-slots // self.page) - len(self.owned[row]))))
        total = sum(count for _, count in counts)
        if total > len(self.free):
            raise RuntimeError(f"the cache has {len(self.free)} free pages, {total} are needed")
        if not total:
            return
        pages = self.free[:-total - 1:-1]
        places = [row % self.rows * self.columns + len(self.owned[row]) + i for row, count in counts for i in range(count)]
        sent = self._sent([places, pages])
        self.tables.view(-1).index_copy_(0, sent[0], sent[1].int())
        del self.free[-total:]
        for row, count in counts:
            self.owned[row].extend(pages[:count])
            del pages[:count]

    def _sent(self, numbers: list[list[int]]) -> Tensor:
        """``numbers`` on the device, in stream order.  A copy from memory that is not pinned would wait for the stream, as would
        assigning a number to an element, for which this class has ``fill_``."""
        given = torch.tensor(numbers, dtype=torch.int64)
        return given.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else given

    def write(self, layer: int, row: int, keys: Tensor, values: Tensor) -> None:
        """Put a prompt's rotated keys and its values, [kv_heads, tokens, head_dim], behind the row's slots in one layer; call
        it for every layer, then ``extend``.  The slots' weights begin at zero."""
        start, tokens = self.held[row], keys.shape[1]
        expected = (self.shape[1], tokens, self.shape[3])
        if tuple(keys.shape) != expected or tuple(values.shape) != expected:
            raise ValueError(f"keys and values are [kv_heads, tokens, head_dim], here {expected}")
        self.reserve(row, start + tokens)
        slot = torch.arange(start, start + tokens, device=self.device)
        at = (self.tables[row].long()[slot // self.page], slice(None), slot % self.page)
        self.k_pages[layer][at] = keys.transpose(0, 1).to(self.dtype)
        self.v_pages[layer][at] = values.transpose(0, 1).to(self.dtype)
        if self.track_weights:
            self.weights[layer][at] = 0.0

    def extend(self, row: int, tokens: int) -> None:
        """Count ``tokens`` slots that ``write`` has filled."""
        self.reserve(row, self.held[row] + tokens)
        self.held[row] += tokens
        self.lengths[row].fill_(self.held[row])

    # -- steps --
    def prepare(self, batch: int) -> None:
        """Before a step of the first ``batch`` rows: every row in use has a page for its next token."""
        if not self._idle:
            self._reserve((row, self.held[row] + 1) for row in range(batch) if self.held[row] >= 0)

    def count(self, batch: int) -> None:
        """The device's part of ``advance``; a captured step contains it."""
        lengths = self.lengths[:batch]
        lengths.add_(lengths >= 0)

    def advance(self, batch: int) -> None:
        """The host's part, after a step or a replay of one."""
        if not self._idle:
            for row in range(batch):
                if self.held[row] >= 0:
                    self.held[row] += 1

    @contextmanager
    def idle(self) -> Iterator[None]:
        """No row is in use meanwhile: steps that warm up or are captured leave the cache as it is."""
        saved = self.lengths.clone()
        self.lengths.fill_(-1)
        self._idle = True
        try:
            yield
        finally:
            self._idle = False
            self.lengths.copy_(saved)

    # -- eviction --
    def evict(self, budget: int, *, sinks: int = 0, recent: int = 0) -> dict[int, list[Tensor]]:
        """Cut every sequence of more than ``budget`` slots down to it: the first ``sinks``, the last ``recent`` and the
        heaviest others of each head and layer stay (``kernels.evict_pages``).  Returns, by row, the kept slots of each layer,
        int32 [kv_heads, budget].  Sequences are moved one after another, so ``budget`` free slots are enough."""
        if not self.track_weights:
            raise ValueError("eviction needs a cache that tracks weights")
        if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"{sinks} first and {recent} last slots do not fit a budget of {budget}")
        kept: dict[int, list[Tensor]] = {}
        need = -(-budget // self.page)
        rows = [row for row in range(self.rows) if self.held[row] > budget]
        if rows and need > len(self.free):
            raise RuntimeError(f"the cache has {len(self.free)} free pages, {need} are needed to evict into")
        for row in rows:
            fresh = [self.free.pop() for _ in range(need)]
            new_tables = self._sent([fresh]).int()
            try:
                kept[row] = [kernels.evict_pages(keys, values, weights, self.tables[row:row + 1], self.lengths[row:row + 1],
                                                 new_tables, budget=budget, sinks=sinks, recent=recent)[0]
                             for keys, values, weights in zip(self.k_pages, self.v_pages, self.weights)]
            except Exception:
                self.free.extend(reversed(fresh))       # the sequence stays where it was
                raise
            self.free.extend(reversed(self.owned[row]))
            self.owned[row], self.held[row] = fresh, budget
            self.tables[row].fill_(-1)
            self.tables[row, :need] = new_tables[0]
            self.lengths[row].fill_(budget)
        return kept


class LogitRules:
    """Penalties, biases and masks of the rows of a batch, on the device for ``kernels.adjust_logits``: histories of up to
    ``capacity`` tokens, up to ``biases`` biased tokens a row, and, with ``vocab``, a mask of allowed tokens."""

    def __init__(self, *, rows: int, capacity: int, biases: int = 0, vocab: int | None = None,
                 device: torch.device | str = "cuda") -> None:
        if rows < 1 or capacity < 1 or biases < 0 or (vocab is not None and vocab < 1):
            raise ValueError("logit rules need rows, a history and a vocabulary of at least one")
        self.rows, self.capacity, self.vocab, self.device = rows, capacity, vocab, torch.device(device)
        full = lambda shape, value, dtype: torch.full(shape, value, dtype=dtype, device=self.device)
        self.tokens = full((rows, capacity), -1, torch.int64)
        self.lengths, self.prompts = full((rows,), 0, torch.int32), full((rows,), 0, torch.int32)
        self.repetition, self.frequency, self.presence = (full((rows,), value, torch.float32) for value in (1.0, 0.0, 0.0))
        self.bias_tokens = full((rows, biases), -1, torch.int32) if biases else None
        self.bias = full((rows, biases), 0.0, torch.float32) if biases else None
        self.mask = full((rows, -(-vocab // 32)), -1, torch.int32) if vocab is not None else None

    def begin(self, row: int, prompt: Sequence[int] = (), *, repetition: float = 1.0, frequency: float = 0.0,
              presence: float = 0.0, bias: Mapping[int, float] | None = None) -> None:
        """The rules of a row's new sequence; its prompt counts for the repetition penalty alone."""
        if len(prompt) > self.capacity:
            raise ValueError(f"a prompt of {len(prompt)} tokens exceeds the history of {self.capacity}")
        if not repetition > 0:
            raise ValueError("the repetition penalty is a positive factor")
        bias = dict(bias or {})
        room = 0 if self.bias is None else self.bias.shape[1]
        if len(bias) > room:
            raise ValueError(f"{len(bias)} biased tokens, room for {room}")
        self.tokens[row, :len(prompt)] = torch.tensor(list(prompt), dtype=torch.int64)
        self.lengths[row] = self.prompts[row] = len(prompt)
        self.repetition[row], self.frequency[row], self.presence[row] = repetition, frequency, presence
        if self.bias is not None:
            self.bias_tokens[row].fill_(-1)
            self.bias_tokens[row, :len(bias)] = torch.tensor(list(bias), dtype=torch.int32)
            self.bias[row, :len(bias)] = torch.tensor(list(bias.values()), dtype=torch.float32)
        self.allow(row, None)

    def allow(self, row: int, tokens: Iterable[int] | None) -> None:
        """Allow a row these tokens only; ``None``: all."""
        if self.mask is None:
            if tokens is not None:
                raise ValueError("these rules have no mask")
            return
        if tokens is None:
            self.mask[row].fill_(-1)
            return
        words = [0] * self.mask.shape[1]
        for token in tokens:
            if not 0 <= token < self.vocab:
                raise ValueError(f"token {token} is not one of {self.vocab}")
            words[token // 32] |= 1 << token % 32
        self.mask[row] = torch.tensor([word - (word >> 31 << 32) for word in words], dtype=torch.int32)

    def observe(self, tokens: Tensor) -> None:
        """Append each row's generated token (int64 [batch]) to its history; a full history takes no more."""
        batch = tokens.shape[0]
        at = self.lengths[:batch].long()
        room = at < self.capacity
        at = at.clamp(max=self.capacity - 1).unsqueeze(1)
        history = self.tokens[:batch]
        history.scatter_(1, at, torch.where(room.unsqueeze(1), tokens.unsqueeze(1), history.gather(1, at)))
        self.lengths[:batch].add_(room)

    @contextmanager
    def idle(self) -> Iterator[None]:
        """What is observed meanwhile is not kept: steps that warm up or are captured leave the histories as they are."""
        saved = self.lengths.clone()
        try:
            yield
        finally:
            self.lengths.copy_(saved)

    def apply(self, logits: Tensor, *, offset: int = 0, best: Tensor | None = None, picked: Tensor | None = None) -> Tensor:
        """``logits`` [batch, width] of the tokens ``offset..offset + width``, adjusted in place by the first ``batch`` rows' rules."""
        batch = logits.shape[0]
        of = lambda table: None if table is None else table[:batch]
        return kernels.adjust_logits(logits, tokens=of(self.tokens), lengths=of(self.lengths), prompts=of(self.prompts),
                                     repetition=of(self.repetition), frequency=of(self.frequency), presence=of(self.presence),
                                     bias_tokens=of(self.bias_tokens), bias=of(self.bias), mask=of(self.mask), offset=offset,
                                     best=best, picked=picked)
