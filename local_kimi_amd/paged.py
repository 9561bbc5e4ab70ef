"""A cache in pages for full attention layers, and the book of who has which page.

:class:`PageBook` hands out pages, counts who shares them and plans the copies that a
shared page or a compaction asks for; it holds numbers alone. :class:`PagedCache` keeps
the pages of all layers with their table and lengths on the device, in the layout that
``kernels.qk_norm_rope_append`` writes and ``kernels.attention_paged`` reads, and carries
a book's copies out with ``kernels.copy_pages``.
"""

from __future__ import annotations

import heapq
from array import array
from collections.abc import Sequence

import torch

from .kernels.paged import PAGE_ROWS_STEP, copy_pages
from .kernels.w4a16 import _on

Copies = tuple[list[int], list[int]]  # pages read, pages written


class PageBook:
    """Sequences of tokens in pages of ``page_rows``, at most ``width`` each.

    A page belongs to every sequence that names it and is free when none does. Only the
    last page of a sequence takes new tokens, so sequences may share all pages until one
    of them grows: ``extend`` then gives it a copy of a last page that is not full. Calls
    that raise change nothing."""

    def __init__(self, pages: int, page_rows: int, sequences: int, width: int) -> None:
        if pages < 0 or page_rows <= 0 or sequences <= 0 or width <= 0:
            raise ValueError("a cache needs sequences, rows and pages a sequence")
        self.page_rows, self.width = page_rows, width
        self.users = [0] * pages                                       # of each page
        self.pages: list[list[int] | None] = [None] * sequences        # of each sequence
        self.lengths = [0] * sequences
        self.changed: set[int] = set()  # sequences whose pages changed; its reader clears it
        self.grown: list[int] = []      # sequences that the last extend gave tokens
        self._free = list(range(pages))  # a heap: the lowest goes first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _check(self, sequence: int) -> list[int]:
        if not 0 <= sequence < len(self.pages) or self.pages[sequence] is None:
            raise ValueError(f"there is no sequence {sequence}")
        return self.pages[sequence]

    def _vacant(self) -> int:
        for i, held in enumerate(self.pages):
            if held is None:
                return i
        raise RuntimeError(f"all {len(self.pages)} sequences are in use")

    def add(self) -> int:
        """A new, empty sequence."""
        i = self._vacant()
        self.pages[i], self.lengths[i] = [], 0
        self.changed.add(i)
        return i

    def fork(self, sequence: int) -> int:
        """A new sequence of the same tokens, on the same pages."""
        held = self._check(sequence)
        i = self._vacant()
        for p in held:
            self.users[p] += 1
        self.pages[i], self.lengths[i] = list(held), self.lengths[sequence]
        self.changed.add(i)
        return i

    def free(self, sequence: int) -> None:
        for p in self._check(sequence):
            self._release(p)
        self.pages[sequence], self.lengths[sequence] = None, 0
        self.grown = [s for s in self.grown if s != sequence]
        self.changed.add(sequence)

    def _release(self, page: int) -> None:
        self.users[page] -= 1
        if self.users[page] == 0:
            heapq.heappush(self._free, page)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self.users[page] = 1
        return page

    def extend(self, sequences: Sequence[int], tokens: Sequence[int]) -> Copies:
        """Room for ``tokens[i]`` more tokens of ``sequences[i]``; returns the copies that
        come before they are written."""
        # (as plain numbers: those of a tensor are equal, and not the same in a set)
        sequences, tokens = list(map(int, sequences)), list(map(int, tokens))
        if len(sequences) != len(tokens) or len(set(sequences)) != len(sequences):
            raise ValueError("extend takes each sequence once, with a number of tokens")
        need, sharers = 0, {}
        for s, n in zip(sequences, tokens):
            held = self._check(s)
            if n < 0:
                raise ValueError(f"sequence {s} cannot grow by {n} tokens")
            total = -(-(self.lengths[s] + n) // self.page_rows)
            if total > self.width:
                raise ValueError(f"sequence {s} would need {total} pages, of at most {self.width}")
            need += total - len(held)
            if n and self.lengths[s] % self.page_rows:
                last = held[-1]
                sharers[last] = sharers.get(last, 0) + 1
        # of a page's users one may write to it, where all of them grow
        need += sum(min(n, self.users[p] - 1) for p, n in sharers.items())
        if need > len(self._free):
            raise RuntimeError(f"{need} pages are needed, {len(self._free)} are free")
        src, dst = [], []
        self.grown = [s for s, n in zip(sequences, tokens) if n]
        for s, n in zip(sequences, tokens):
            held = self.pages[s]
            if n and self.lengths[s] % self.page_rows and self.users[held[-1]] > 1:
                src.append(held[-1])
                self._release(held[-1])
                held[-1] = self._take()
                dst.append(held[-1])
                self.changed.add(s)
            self.lengths[s] += n
            while len(held) * self.page_rows < self.lengths[s]:
                held.append(self._take())
                self.changed.add(s)
        return src, dst

    def compact(self) -> Copies:
        """The pages in use become the lowest ones; returns the copies that move them."""
        used = sum(1 for n in self.users if n)
        src = [p for p in range(used, len(self.users)) if self.users[p]]
        dst = [p for p in range(used) if not self.users[p]]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.users[a], self.users[b] = 0, self.users[a]
        self.pages = [held if held is None else [to.get(p, p) for p in held] for held in self.pages]
        self._free = list(range(used, len(self.users)))
        if to:
            self.changed.update(i for i, held in enumerate(self.pages) if held)
        return src, dst


class PagedCache:
    """Keys and values of up to ``sequences`` sequences of ``capacity`` tokens each, in
    ``pages`` pages that the ``layers`` full attention layers use alike.

    ``k_pages[layer]`` and ``v_pages[layer]`` [pages, rows, kv_heads, d], ``page_table``
    [sequences, pages a sequence], ``lengths`` and ``step_lengths`` [sequences] stay where
    they are, so that a captured graph finds later contents there. ``step_lengths`` are the
    lengths of the sequences that the last ``extend`` gave tokens, and 0 for the others.

    A decode step over all sequences is ``extend`` by one token for each that takes part, then
    per layer ``qk_norm_rope_append`` and ``attention_paged`` on ``page_table`` and
    ``step_lengths``: a sequence that did not grow, or is not in use, is not written and
    attends to nothing. (By ``lengths`` its row would replace its last token, also in a page that
    a fork shares.) ``rows_of`` picks the rows of some sequences, by ``lengths``. Copies
    and uploads are issued on the current stream, and nothing waits for them; calls that make
    them are refused while it is captured."""

    def __init__(self, pages: int, sequences: int, capacity: int, *, layers: int, kv_heads: int,
                 d_qk: int, d_v: int, page_rows: int = 64, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> None:
        if page_rows <= 0 or page_rows % PAGE_ROWS_STEP:
            raise ValueError(f"a page must have a multiple of {PAGE_ROWS_STEP} rows, got {page_rows}")
        self.book = PageBook(pages, page_rows, sequences, -(-capacity // page_rows))

        def made(d):
            return torch.zeros((layers, pages, page_rows, kv_heads, d), dtype=dtype, device=device)

        self.k_pages, self.v_pages = list(made(d_qk)), list(made(d_v))
        self._table = torch.full((sequences, self.book.width), -1, dtype=torch.int32)
        self.page_table = self._table.to(device, copy=True)
        self._counts = torch.zeros((2, sequences), dtype=torch.int32, device=device)
        self.lengths, self.step_lengths = self._counts

    def _check_stream(self) -> None:
        """Before anything changes: a replay would upload from memory that is long free."""
        if not self.lengths.is_cuda:
            return
        with _on(self.lengths.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a paged cache is extended, forked, freed from, compacted and asked "
                                   "for rows outside the captured graph")

    def _upload(self, target: torch.Tensor, values: torch.Tensor) -> None:
        # from pinned memory of its own, so that the copy takes its turn on the stream
        target.copy_(values.pin_memory() if target.is_cuda else values, non_blocking=True)

    def _carry_out(self, copies: Copies) -> None:
        if copies[0]:
            copy_pages([*self.k_pages, *self.v_pages], *copies)
        if self.book.changed:
            for i in self.book.changed:
                held = self.book.pages[i] or []
                self._table[i].fill_(-1)
                self._table[i, :len(held)] = torch.tensor(held, dtype=torch.int32)
            self.book.changed.clear()
            self._upload(self.page_table, self._table)
        step = [0] * len(self.book.lengths)
        for i in self.book.grown:
            step[i] = self.book.lengths[i]
        counts = torch.frombuffer(array("i", self.book.lengths + step), dtype=torch.int32)
        self._upload(self._counts, counts.view(2, -1))

    def add(self) -> int:
        """A new, empty sequence."""
        return self.book.add()

    def extend(self, sequences: Sequence[int], tokens: Sequence[int]) -> None:
        """Room for more tokens, counted in ``lengths``: the next calls on the cache write
        and read them as the sequences' new ones. Shared last pages are copied first."""
        self._check_stream()
        self._carry_out(self.book.extend(sequences, tokens))

    def fork(self, sequence: int) -> int:
        """A new sequence that starts with the tokens of ``sequence``, on its pages."""
        self._check_stream()
        i = self.book.fork(sequence)
        self._carry_out(([], []))
        return i

    def free(self, sequence: int) -> None:
        self._check_stream()
        self.book.free(sequence)
        self._carry_out(([], []))

    def compact(self) -> int:
        """Moves the pages in use to the front of the tensors; returns how many moved."""
        self._check_stream()
        copies = self.book.compact()
        self._carry_out(copies)
        return len(copies[0])

    def rows_of(self, sequences: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor]:
        """``page_table`` and ``lengths`` of these sequences, in this order (copies); one that is
        not in use has length 0 and no pages."""
        self._check_stream()
        sequences = [int(s) for s in sequences]
        for s in sequences:
            if not 0 <= s < len(self.book.pages):  # (an index on the device would fault there)
                raise ValueError(f"there is no sequence {s} of {len(self.book.pages)}")
        at = torch.empty(len(sequences), dtype=torch.int64, device=self.lengths.device)
        self._upload(at, torch.tensor(sequences, dtype=torch.int64))
        return self.page_table[at], self.lengths[at]
