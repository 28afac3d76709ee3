"""The host's side of a 4-bit paged cache: which pages are free, whose the others are, and what a step
over a batch of sequences has to tell the kernels (radiance_kv4.qk_norm_rope_append and attention).

  pool = PagePool(new_cache(pages, kv_heads, page, head_size, layers=L))
  a = pool.add()
  step = pool.extend([a], [prompt_tokens])       # pages for the new tokens; slots, lengths, tables
  for layer in ...:                              # append at step.slots, attend over step.page_table
  b = pool.fork(a)                               # shares a's pages; copied only when written
  step = pool.extend([a, b], [1, 1])
  pool.truncate(b, length)                       # drops rejected tokens
  pool.free(a)
  pool.compact()                                 # pages in use to the front

Not thread-safe: one pool belongs to one scheduler. Kernels of earlier steps may still run while the
pool changes: pages are written by later launches of the same stream only.
"""
from __future__ import annotations

import heapq
from typing import NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import radiance_kv4 as _kv4


class Step(NamedTuple):
    """A batch's new tokens, for every layer: sequence b's are rows q_starts[b] .. q_starts[b + 1] - 1."""
    slots: torch.Tensor        # int64 [total], where their keys and values go
    positions: torch.Tensor    # int64 [total], their places in their sequences
    page_table: torch.Tensor   # int32 [batch, pages of the longest]
    seq_lens: torch.Tensor     # int32 [batch], the new ones among them
    q_starts: torch.Tensor     # int32 [batch + 1]
    max_q: int
    max_len: int

    @property
    def attention(self):
        """What radiance_kv4.attention takes after q and the cache."""
        return self.page_table, self.seq_lens, self.q_starts, self.max_q, self.max_len


def _fail(what: str):
    raise RuntimeError(f"[radiance.kv4] PagePool: {what}")


class _Sequence:
    __slots__ = ("pages", "length")

    def __init__(self, pages, length):
        self.pages, self.length = pages, length


class PagePool:
    """Pages of `cache` ([pages, ...] or [layers, pages, ...] of new_cache), lowest free page first."""

    def __init__(self, cache: torch.Tensor):
        if cache.dim() not in (4, 5):
            _fail(f"cache must be one of new_cache, got {tuple(cache.shape)}")
        self.cache = cache
        self.pages, self.page = cache.shape[-4], cache.shape[-2] * _kv4.GROUP
        self._free = list(range(self.pages))       # a heap
        self._refs = [0] * self.pages              # sequences that a page belongs to
        self._sequences: dict[int, _Sequence] = {}
        self._next = 0

    # ---- what there is
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._get(sequence).length

    def pages_of(self, sequence: int) -> list[int]:
        return list(self._get(sequence).pages)

    def _get(self, sequence: int) -> _Sequence:
        s = self._sequences.get(sequence)
        if s is None:
            _fail(f"no sequence {sequence}")
        return s

    # ---- sequences
    def add(self) -> int:
        """A new, empty sequence."""
        self._sequences[self._next] = _Sequence([], 0)
        self._next += 1
        return self._next - 1

    def fork(self, sequence: int, length: Optional[int] = None) -> int:
        """A new sequence of the first `length` tokens (all by default) of another. Their pages are
        shared; extend() copies a page that is not full when one of its sequences goes on."""
        s = self._get(sequence)
        length = s.length if length is None else int(length)
        if not 0 <= length <= s.length:
            _fail(f"fork of {length} tokens of the {s.length} of sequence {sequence}")
        pages = s.pages[:-(-length // self.page)]
        for p in pages:
            self._refs[p] += 1
        new = self.add()
        self._sequences[new] = _Sequence(pages, length)
        return new

    def free(self, sequence: int) -> None:
        self._drop(self._get(sequence).pages)
        del self._sequences[sequence]

    def truncate(self, sequence: int, length: int) -> None:
        """Keeps the first `length` tokens of a sequence (after drafted tokens were rejected)."""
        s = self._get(sequence)
        if not 0 <= length <= s.length:
            _fail(f"truncate to {length} tokens of the {s.length} of sequence {sequence}")
        keep = -(-int(length) // self.page)
        self._drop(s.pages[keep:])
        del s.pages[keep:]
        s.length = int(length)

    def _drop(self, pages) -> None:
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)

    # ---- steps
    def extend(self, sequences: Sequence[int], counts: Sequence[int]) -> Step:
        """Room for counts[i] more tokens of each sequence, and the step that fills it. The last, partly
        filled page of a sequence that shares it is copied first (in all layers, one launch, on the
        current stream). RuntimeError where the free pages do not suffice; what fails changes nothing."""
        if len(sequences) != len(counts) or len(set(sequences)) != len(sequences):
            _fail(f"extend of sequences {list(sequences)} by {list(counts)}")
        batch = [self._get(i) for i in sequences]
        counts = [int(n) for n in counts]
        if counts and min(counts) < 0:
            _fail(f"extend by {counts} tokens")
        copies, shared, need = [], {}, 0
        for s, n in zip(batch, counts):
            copy = False
            if n and s.length % self.page:
                last = s.pages[-1]
                left = shared.setdefault(last, self._refs[last])
                copy = left > 1
                shared[last] = left - 1 if copy else left
            copies.append(copy)
            need += -(-(s.length + n) // self.page) - len(s.pages) + copy
        if need > len(self._free):
            _fail(f"{need} pages needed, {len(self._free)} of {self.pages} free")
        pairs, taken, old = [], [], []

        def take():
            taken.append(heapq.heappop(self._free))
            self._refs[taken[-1]] = 1
            return taken[-1]
        try:
            for s, n, copy in zip(batch, counts, copies):
                old.append((s, len(s.pages), s.length, s.pages[-1] if copy else None))
                if copy:
                    pairs.append((s.pages[-1], take()))
                    self._refs[s.pages[-1]] -= 1
                    s.pages[-1] = taken[-1]
                s.length += n
                while len(s.pages) * self.page < s.length:
                    s.pages.append(take())
            if pairs:
                _kv4.move_pages(self.cache, torch.tensor(pairs, dtype=torch.int32))
            return self._step(batch, counts)
        except Exception:               # of the launch or an allocation
            for s, pages, length, shared_page in old:
                del s.pages[pages:]
                s.length = length
                if shared_page is not None:
                    s.pages[-1] = shared_page
                    self._refs[shared_page] += 1
            for p in taken:
                self._refs[p] = 0
                heapq.heappush(self._free, p)
            raise

    def _step(self, batch, counts) -> Step:
        # One host buffer and one copy: slots and positions (8 bytes each), then the int32 parts.
        total, B = sum(counts), len(batch)
        cols = max((len(s.pages) for s in batch), default=0)
        sizes = [2 * total, 2 * total, B * cols, B, B + 1]
        cuda = self.cache.device.type == "cuda"
        host = torch.empty(sum(sizes), dtype=torch.int32, pin_memory=cuda)
        at = np.cumsum([0] + sizes)
        part = [host.numpy()[a:b] for a, b in zip(at[:-1], at[1:])]
        slots, positions = part[0].view(np.int64), part[1].view(np.int64)
        table = part[2].reshape(B, cols)
        done = 0
        part[4][0] = 0
        for b, (s, n) in enumerate(zip(batch, counts)):
            table[b, :len(s.pages)] = s.pages
            table[b, len(s.pages):] = -1
            place = np.arange(s.length - n, s.length, dtype=np.int64)
            positions[done:done + n] = place
            slots[done:done + n] = table[b].astype(np.int64)[place // self.page] * self.page \
                + place % self.page
            done += n
            part[3][b], part[4][b + 1] = s.length, done
        dev = host.to(self.cache.device, non_blocking=True)
        p = [dev[a:b] for a, b in zip(at[:-1], at[1:])]
        return Step(p[0].view(torch.int64), p[1].view(torch.int64), p[2].view(B, cols), p[3], p[4],
                    max(counts, default=0), max((s.length for s in batch), default=0))

    # ---- compaction
    def compact(self, page_table: Optional[torch.Tensor] = None) -> int:
        """Moves the pages in use to the front of the cache, in all layers, and returns how many moved.
        Steps made before are void; a page table that outlives them (a captured graph's) is remapped
        on the device where it is given."""
        used = [p for p in range(self.pages) if self._refs[p]]
        n = len(used)
        holes = [p for p in range(n) if not self._refs[p]]
        moves = dict(zip([p for p in used if p >= n], holes))
        if not moves:
            return 0
        _kv4.move_pages(self.cache, torch.tensor(list(moves.items()), dtype=torch.int32), page_table)
        for s in self._sequences.values():
            s.pages = [moves.get(p, p) for p in s.pages]
        for a, b in moves.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(n, self.pages))    # ascending: a heap
        return len(moves)
