"""A paged key-value cache for serving: which pages a sequence has (host), and
the pools that hold them (GPU).

``PageAllocator`` is the bookkeeping alone, in plain Python: sequences grow by
whole pages, forks share pages until one of them writes (copy on write),
freed pages are reused, and compaction moves the live pages to the front.
Whatever has to move in memory comes back as (source, destination) page
numbers.  ``PagedKVCache`` adds the pools of all layers and carries the moves
out with one ``kv_pages_copy`` launch.

    cache = PagedKVCache(num_layers, num_pages, page_size, num_kv_heads, head_dim)
    a = cache.new_sequence()
    step = cache.extend([a], [len(prompt)])     # pages for the new tokens
    for layer ...:
        cache.write(layer, step, k, v)          # [tokens, kv_heads, head_dim]
        out = cache.prompt_attention(step, q, k, v)     # a fresh prompt
    b = cache.fork(a)                           # shares a's pages
    step = cache.extend([a, b], [1, 1])
    for layer ...:
        cache.write(layer, step, k, v)
        out = cache.decode_attention(layer, step, q)    # one token a sequence
    cache.free(b)
    cache.compact()

A step's device arrays belong to that step; all work goes to the current
stream, so steps follow one another without synchronisation.  The reference
has no counterpart (its decode kernels take one contiguous cache).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch


class OutOfPages(RuntimeError):
    """There are not enough free pages; nothing has been changed."""


class PageAllocator:
    """Pages of sequences, with sharing.  No tensors, no GPU."""

    def __init__(self, num_pages: int, page_size: int):
        if num_pages <= 0 or page_size <= 0:
            raise ValueError(f"num_pages ({num_pages}) and page_size ({page_size}) must be positive")
        self.num_pages = num_pages
        self.page_size = page_size
        self._uses = [0] * num_pages
        self._free = list(range(num_pages - 1, -1, -1))  # the lowest page is taken first
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> list[int]:
        return list(self._pages)

    def length(self, seq: int) -> int:
        return self._length[self._known(seq)]

    def pages(self, seq: int) -> list[int]:
        return list(self._pages[self._known(seq)])

    def _known(self, seq: int) -> int:
        if seq not in self._pages:
            raise KeyError(f"no sequence {seq!r} in the cache")
        return seq

    def new_sequence(self) -> int:
        seq = self._next
        self._next += 1
        self._pages[seq] = []
        self._length[seq] = 0
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens, on the same pages."""
        pages = self._pages[self._known(seq)]
        child = self.new_sequence()
        self._pages[child] = list(pages)
        self._length[child] = self._length[seq]
        for p in pages:
            self._uses[p] += 1
        return child

    def free(self, seq: int) -> None:
        for p in self._pages.pop(self._known(seq)):
            self._drop(p)
        del self._length[seq]

    def _drop(self, page: int) -> None:
        self._uses[page] -= 1
        if self._uses[page] == 0:
            self._free.append(page)

    def _take(self) -> int:
        page = self._free.pop()
        self._uses[page] = 1
        return page

    def extend(self, seqs: list[int], counts: list[int]) -> list[tuple[int, int]]:
        """Room for counts[i] more tokens of seqs[i]; the pages to copy first.

        The page that a sequence goes on writing to is copied if another one
        shares it.  Raises OutOfPages, with nothing changed, if the pages do
        not suffice."""
        if len(seqs) != len(counts):
            raise ValueError("seqs and counts must have the same length")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence can be extended once a step")
        if any(n < 0 for n in counts):
            raise ValueError("counts must not be negative")
        size = self.page_size
        need, uses = 0, {}
        for seq, n in zip(seqs, counts):
            pages, length = self._pages[self._known(seq)], self._length[seq]
            if n and length % size:
                last = pages[-1]
                if uses.setdefault(last, self._uses[last]) > 1:
                    uses[last] -= 1
                    need += 1
            need += -(-(length + n) // size) - len(pages)
        if need > len(self._free):
            raise OutOfPages(f"{need} pages are needed, {len(self._free)} of {self.num_pages} "
                             "are free")
        moves = []
        for seq, n in zip(seqs, counts):
            pages, length = self._pages[seq], self._length[seq]
            if n and length % size and self._uses[pages[-1]] > 1:
                page = self._take()
                moves.append((pages[-1], page))
                self._drop(pages[-1])
                pages[-1] = page
            while len(pages) * size < length + n:
                pages.append(self._take())
            self._length[seq] = length + n
        return moves

    def withdraw(self, seqs: list[int], counts: list[int]) -> None:
        """Takes the last counts[i] tokens of seqs[i] back: those of a step that failed."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs):
            raise ValueError("withdraw: one count for each of different sequences")
        for seq, n in zip(seqs, counts):
            if not 0 <= n <= self._length[self._known(seq)]:
                raise ValueError(f"withdraw: {n} tokens of a sequence of {self._length[seq]}")
        for seq, n in zip(seqs, counts):
            self._length[seq] -= n
            pages = self._pages[seq]
            while (len(pages) - 1) * self.page_size >= self._length[seq] and pages:
                self._drop(pages.pop())

    def compact(self) -> list[tuple[int, int]]:
        """Renumbers the live pages to 0 .. n - 1; the pages to move."""
        live = sum(u > 0 for u in self._uses)
        holes = [p for p in range(live) if self._uses[p] == 0]
        high = [p for p in range(live, self.num_pages) if self._uses[p] > 0]
        to = dict(zip(high, holes))
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._uses[a], self._uses[b] = 0, self._uses[a]
        self._free = list(range(self.num_pages - 1, live - 1, -1))
        return list(to.items())


@dataclass
class Step:
    """Tokens that one step adds: device arrays for its launches."""
    seqs: list
    counts: list
    page_table: torch.Tensor    # int32 [batch, pages of the longest]
    start_lens: torch.Tensor    # int32 [batch], tokens before the step
    seq_lens: torch.Tensor      # int32 [batch], tokens after it
    cu_seqlens: torch.Tensor    # int32 [batch + 1], the new tokens' rows
    positions: torch.Tensor     # int32 [tokens], the new tokens' positions
    max_count: int
    fresh: bool                 # every sequence was empty before


class PagedKVCache(PageAllocator):
    """The pools of num_layers layers, [num_pages, page_size, num_kv_heads,
    head_dim] for K and for V each, and their sequences."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int,
                 head_dim: int, dtype=torch.bfloat16, device="cuda"):
        super().__init__(num_pages, page_size)
        from src.load_gqa_attention import gqa_attention_cuda

        self._ops = gqa_attention_cuda
        self.device = torch.device(device)
        shape = (num_pages, page_size, num_kv_heads, head_dim)
        self.k_pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v_pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.scale = 1.0 / math.sqrt(head_dim)

    def _move(self, moves: list[tuple[int, int]]) -> None:
        if moves:
            self._ops.kv_pages_copy(self.k_pages + self.v_pages, [a for a, _ in moves],
                                    [b for _, b in moves])

    def extend(self, seqs: list[int], counts: list[int]) -> Step:
        """Room for counts[i] more tokens of seqs[i], pages shared with other
        sequences copied where the step writes to them."""
        self._move(super().extend(seqs, counts))
        try:
            return self._step(seqs, counts)
        except Exception:  # no memory for the step's arrays
            self.withdraw(seqs, counts)
            raise

    def _step(self, seqs: list[int], counts: list[int]) -> Step:
        after = [self._length[s] for s in seqs]
        before = [a - n for a, n in zip(after, counts)]
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        positions = [p for b, a in zip(before, after) for p in range(b, a)]
        width = max([len(self._pages[s]) for s in seqs] + [1])
        table = [p for s in seqs for p in
                 self._pages[s] + [-1] * (width - len(self._pages[s]))]
        # One upload for all of it.
        parts = [table, before, after, cu, positions]
        host = torch.tensor([x for part in parts for x in part], dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        table, before, after, cu, positions = host.to(self.device, non_blocking=True).split(
            [len(part) for part in parts])
        return Step(list(seqs), list(counts), table.view(len(seqs), width), before, after, cu,
                    positions, max(list(counts) + [0]),
                    all(self._length[s] == n for s, n in zip(seqs, counts)))

    def write(self, layer: int, step: Step, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's new keys and values, [tokens, num_kv_heads, head_dim], into the pages."""
        self._ops.kv_cache_append(k, v, self.k_pages[layer], self.v_pages[layer], step.page_table,
                                  step.start_lens, step.cu_seqlens)

    def prompt_attention(self, step: Step, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         scale: float | None = None) -> torch.Tensor:
        """Causal attention of a step of fresh prompts, packed: q [tokens, heads, head_dim]."""
        if not step.fresh:
            raise ValueError("prompt_attention: a sequence of this step had tokens before it")
        return self._ops.gqa_prompt_attention(q, k, v, step.cu_seqlens, step.max_count,
                                              self.scale if scale is None else scale)

    def decode_attention(self, layer: int, step: Step, q: torch.Tensor,
                         scale: float | None = None) -> torch.Tensor:
        """Attention of one new token a sequence over its cached tokens, itself
        (written before) among them: q [batch, heads, head_dim]."""
        if any(n != 1 for n in step.counts):
            raise ValueError("decode_attention: the step must add one token to each sequence")
        return self._ops.gqa_paged_decode(q, self.k_pages[layer], self.v_pages[layer],
                                          step.page_table, step.seq_lens,
                                          self.scale if scale is None else scale)

    def compact(self) -> int:
        """Moves the live pages to the front of the pools; how many moved.
        Steps made before are void."""
        moves = super().compact()
        self._move(moves)
        return len(moves)
