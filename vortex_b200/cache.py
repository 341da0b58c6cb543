"""Inference-cache containers with the reference's names, fields and layout
(``vortex/model/cache.py:12-61``).  The engine reads and writes exactly these
dictionaries, keyed by layer index:

* ``fir_state_dict[layer]``        [B, 3D, K3-1]  last featurizer inputs, packed-channel order
* ``fir_inner_state_dict[layer]``  [B, D, K-1]    last k*v samples, oldest first (FIR layers)
* ``state_dict[layer]``            [B, D, S] fp32 modal state, residues not applied (long layers)

Prefill writes the FIR caches in the activation dtype; every decode step returns them in fp32
(``vortex/model/engine.py:427-449``).
"""
import contextlib
import heapq
from dataclasses import dataclass, field
from typing import Optional, Sequence

import torch
from torch import Tensor


@dataclass
class InferenceParams:
    """Attention KV-cache bookkeeping (kept for interface parity; not touched by the Hyena engine).  ``PagedKVCache`` below
    is what ``AttentionInferenceEngine`` keeps its keys and values in."""

    max_seqlen: int
    max_batch_size: int
    seqlen_offset: int = 0
    batch_size_offset: int = 0
    key_value_memory_dict: dict = field(default_factory=dict)
    lengths_per_sample: Optional[Tensor] = None

    def reset(self, max_seqlen, max_batch_size):
        self.max_seqlen, self.max_batch_size, self.seqlen_offset = max_seqlen, max_batch_size, 0
        if self.lengths_per_sample is not None:
            self.lengths_per_sample.zero_()


@dataclass
class HyenaCascadeIIRInferenceParams:
    """Caches of the long (modal IIR) Hyena layers."""

    fir_filter_length: int = 3
    state_dim: int = 16
    seqlen_offset: int = 0
    fir_state_dict: dict = field(default_factory=dict)
    state_dict: dict = field(default_factory=dict)

    def reset(self):
        self.fir_filter_length, self.state_dim, self.seqlen_offset = 3, 16, 0


@dataclass
class HyenaCascadeFIRInferenceParams:
    """Caches of the short and medium (explicit FIR) Hyena layers."""

    fir_filter_length: int = 3
    fir_inner_filter_length: int = 4
    seqlen_offset: int = 0
    fir_inner_state_dict: dict = field(default_factory=dict)
    fir_state_dict: dict = field(default_factory=dict)
    state_dict: dict = field(default_factory=dict)

    def reset(self):
        self.fir_filter_length, self.fir_inner_filter_length, self.seqlen_offset = 3, 4, 0


class PagedKVCache:
    """Keys and values of a stack's attention layers, in pages of ``page_size`` tokens that the sequences share.

    ``k[layer]``, ``v[layer]``: pools [num_pages, page_size, num_heads, head_dim].  A page number means the same page in
    every pool: a sequence holds ``ceil(length / page_size)`` of them, listed in its row of ``block_table`` (int32
    [max_sequences, max_length / page_size], -1 behind the last).  The numbers are kept on the host, where the planning is
    done; the device holds the table, and for the step at work ``positions`` (int32 [max_sequences], the new token's, -1
    where a row has none) and ``lengths`` (its keys, the new one included, 0 where a row has none).  These tensors keep their
    addresses: a captured decode step follows what ``step`` puts there before each replay.

    ``open`` / ``extend`` / ``step`` / ``free`` change the bookkeeping on the host and upload what changed on the current
    stream; ``fork`` and ``compact`` copy pages as well (``attn_ops.copy_pages``).  Under stream capture all but ``open`` are
    refused: their uploads would not be part of the graph.  A call that raises has changed nothing (bookkeeping follows the
    uploads; one that fails after another is done takes that back).  Not thread-safe."""

    def __init__(self, layers, num_pages, page_size, num_heads, head_dim, *, max_sequences, max_length, device="cuda",
                 dtype=torch.bfloat16):
        if min(layers, num_pages, page_size, num_heads, head_dim, max_sequences, max_length) < 1:
            raise ValueError("a paged cache needs at least one of everything")
        shape = (num_pages, page_size, num_heads, head_dim)
        self.k = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(layers)]
        self.v = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(layers)]
        self.page_size, self.num_pages, self.max_length = page_size, num_pages, max_length
        width = -(-max_length // page_size)
        self.block_table = torch.full((max_sequences, width), -1, device=device, dtype=torch.int32)
        self._step = torch.zeros(2, max_sequences, device=device, dtype=torch.int32)
        self._step[0] = -1
        self.positions, self.lengths = self._step[0], self._step[1]
        self._at_work = ([-1] * max_sequences, [0] * max_sequences)                  # the host's copy of these two
        self._table = torch.full((max_sequences, width), -1, device="cpu", dtype=torch.int32)      # the host's copy
        self._pages: list[Optional[list[int]]] = [None] * max_sequences              # of each open row
        self._length = [0] * max_sequences
        self._users = [0] * num_pages                                                # rows that hold a page
        self._unused = list(range(num_pages))                                        # a heap: lowest numbers first

    # -- what is there
    def length(self, row: int) -> int:
        self._check(row)
        return self._length[row]

    def pages(self, row: int) -> list[int]:
        self._check(row)
        return list(self._pages[row])

    @property
    def unused_pages(self) -> int:
        return len(self._unused)

    def _check(self, row):
        if not 0 <= row < len(self._pages) or self._pages[row] is None:
            raise ValueError(f"row {row} holds no sequence")

    def _take(self, count: int) -> list[int]:
        """The lowest unused pages, out of the heap but not yet anyone's."""
        if count > len(self._unused):
            raise RuntimeError(f"{count} page{'s' if count > 1 else ''} needed, {len(self._unused)} unused")
        return [heapq.heappop(self._unused) for _ in range(count)]

    def _put_back(self, pages) -> None:
        for page in pages:
            heapq.heappush(self._unused, page)

    def _not_captured(self) -> None:
        if self.block_table.is_cuda:
            with torch.cuda.device(self.block_table.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("a paged cache cannot be changed under stream capture")

    def _upload(self, rows: Sequence[int]) -> None:
        """The rows' part of the table, in one copy.  (From pageable memory, which CUDA has read when the call returns: the
        host's copy may change afterwards.  Whether the driver waits for the stream meanwhile is up to it.)"""
        if rows:
            lo, hi = min(rows), max(rows) + 1
            self.block_table[lo:hi].copy_(self._table[lo:hi], non_blocking=True)

    def _upload_step(self, at_work) -> None:
        self._step.copy_(torch.tensor(at_work, device="cpu", dtype=torch.int32), non_blocking=True)

    def _change_table(self, entries, then=None):
        """Table entries {row: (first entry, pages)} on the host and the device, then whatever else the call has to upload;
        returns what that returns.  If any of it raises, the table is as it was."""
        rows = [row for row, (_, pages) in entries.items() if len(pages)]
        before, done = [], False
        try:
            for row in rows:
                first, pages = entries[row]
                part = self._table[row, first:first + len(pages)]
                before.append((part, part.clone()))
                part[:] = torch.tensor(pages, device="cpu", dtype=torch.int32)
            self._upload(rows)
            done = True
            return then() if then else None
        except BaseException:
            for part, was in before:
                part[:] = was
            if done:
                with contextlib.suppress(Exception):
                    self._upload(rows)
            raise

    # -- sequences
    def open(self) -> int:
        """An empty sequence; returns its row."""
        for row, pages in enumerate(self._pages):
            if pages is None:
                self._pages[row], self._length[row] = [], 0
                return row
        raise RuntimeError(f"all {len(self._pages)} rows hold sequences")

    def _grow(self, rows, counts, upload):
        """Room for counts[i] more tokens of rows[i]; returns what ``upload`` returns, which is called when the table is there."""
        self._not_captured()
        if len(set(rows)) != len(rows):
            raise ValueError("a row occurs twice")
        need = []
        for row, n in zip(rows, counts):
            self._check(row)
            if n < 0 or self._length[row] + n > self.max_length:
                raise ValueError(f"row {row}: {self._length[row]} + {n} tokens of at most {self.max_length}")
            need.append(-(-(self._length[row] + n) // self.page_size) - len(self._pages[row]))
        taken = self._take(sum(need))
        new, at = {}, 0
        for row, n in zip(rows, need):
            new[row] = (len(self._pages[row]), taken[at:at + n])
            at += n
        try:
            made = self._change_table(new, upload)
        except BaseException:
            self._put_back(taken)
            raise
        for row, n in zip(rows, counts):
            self._length[row] += n
            self._pages[row] += new[row][1]
        for page in taken:
            self._users[page] = 1
        return made

    def extend(self, rows: Sequence[int], counts: Sequence[int]):
        """Room for ``counts[i]`` new tokens of sequence ``rows[i]``; returns their positions and rows (int32, on the device),
        all of the first sequence's, then the second's: what ``attn_ops.rotary_append`` takes for a (ragged) prompt."""
        rows, counts = list(rows), list(counts)
        if len(rows) != len(counts):
            raise ValueError("one count for every row")
        first = [self.length(row) for row in rows]

        def upload():
            both = torch.empty(2, sum(counts), device="cpu", dtype=torch.int32)
            at = 0
            for row, start, n in zip(rows, first, counts):
                both[0, at:at + n] = torch.arange(start, start + n, device="cpu", dtype=torch.int32)
                both[1, at:at + n] = row
                at += n
            return both.to(self.block_table.device, non_blocking=True)

        both = self._grow(rows, counts, upload)
        return both[0], both[1]

    def step(self, rows: Optional[Sequence[int]] = None) -> None:
        """Room for one new token of each of ``rows`` (None: every open sequence); ``positions`` and ``lengths`` say so to
        the decode step that follows."""
        rows = [r for r, p in enumerate(self._pages) if p is not None] if rows is None else list(rows)

        def upload():
            positions, lengths = [-1] * len(self._pages), [0] * len(self._pages)
            for row in rows:
                positions[row], lengths[row] = self._length[row], self._length[row] + 1
            self._upload_step((positions, lengths))
            return positions, lengths

        self._at_work = self._grow(rows, [1] * len(rows), upload)

    def fork(self, row: int) -> int:
        """A sequence that begins as a copy of ``row``: full pages are shared, an open last page is copied in every pool.
        Returns its row.  What it holds is what the stream has stored by then: tokens that ``extend`` or ``step`` made room
        for are stored first."""
        self._not_captured()
        self._check(row)
        pages = list(self._pages[row])
        own = self._take(1) if self._length[row] % self.page_size else []
        child = None
        try:
            child = self.open()
            if own:
                from . import attn_ops

                attn_ops.copy_pages(self.k + self.v, pages[-1:], own)
                pages[-1:] = own
            self._change_table({child: (0, pages)})
        except BaseException:
            self._put_back(own)
            if child is not None:
                self._pages[child] = None
            raise
        for page in pages:
            self._users[page] += 1
        self._pages[child], self._length[child] = pages, self._length[row]
        return child

    def free(self, row: int) -> None:
        """Ends a sequence; pages that no other sequence holds are unused again, and the step at work, if the row is in it, goes
        on without."""
        self._not_captured()
        self._check(row)
        positions, lengths = map(list, self._at_work)
        in_step = lengths[row] > 0
        positions[row], lengths[row] = -1, 0
        self._change_table({row: (0, [-1] * len(self._pages[row]))}, (lambda: self._upload_step((positions, lengths))) if in_step else None)
        self._at_work = positions, lengths
        for page in self._pages[row]:
            self._users[page] -= 1
            if self._users[page] == 0:
                heapq.heappush(self._unused, page)
        self._pages[row], self._length[row] = None, 0

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers and returns how many there are: what lies behind them in the pools
        is free to be given back or reused."""
        from . import attn_ops

        self._not_captured()
        used = self.num_pages - len(self._unused)
        src = [p for p in range(used, self.num_pages) if self._users[p]]
        dst = sorted(p for p in self._unused if p < used)
        if not src:
            return used
        attn_ops.copy_pages(self.k + self.v, src, dst)
        to = dict(zip(src, dst))
        moved = {row: [to.get(p, p) for p in pages] for row, pages in enumerate(self._pages) if pages and any(p in to for p in pages)}
        self._change_table({row: (0, pages) for row, pages in moved.items()})
        for row, pages in moved.items():
            self._pages[row] = pages
        for a, b in to.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._unused = list(range(used, self.num_pages))
        return used
