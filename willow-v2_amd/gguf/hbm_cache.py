"""Every sequence's keys and values resident in device memory as 8-bit pages, in place of the reference's bf16 cache tensors
(one per layer, growing in blocks of 256 positions for one conversation; engines/base.py:213-216,348-358). 288 GB of HBM
holds the pages of many conversations: at Qwen3.6-35B-A3B's two kv heads of 256 a token takes 1 KB a layer.

Pages belong to sequences through a page table kept on the host (PageBook): sequences share the pages they have in common
after a fork, a page that is about to be written while shared is copied first, freed pages are used again, and compact() moves
what is live to the lowest page numbers. The lowest free page is always taken first, so the same calls give the same pages.

    cache = HBMKVCache(layers=10, pages=4096, kv_heads=2, head_dim=256)
    seq = cache.new()
    step = cache.step([seq], [tokens])                        # room for the new tokens, on the GPU what the kernels read
    for layer in range(10):
        cache.append(layer, step, k, v)                       # k, v bf16 [tokens, kv_heads, head_dim]
        out = cache.attend(layer, step, q)                    # q bf16 [tokens, heads, head_dim]

Calls may come on any streams: the cache orders its work as its calls are (_StreamOrder). A captured graph's replays it does
not see: replay on the stream on which refresh() was called for it.
"""
import contextlib
import heapq
from dataclasses import dataclass, field

import numpy as np
import torch

from .hip import KVPages, kv_append, kv_attend, kv_copy


class OutOfPages(RuntimeError):
    """A step needs more pages than are free; nothing was changed."""


def _whole(n) -> int:
    """A number of tokens as an int; a fraction of one is refused."""
    if type(n) is int:
        return n
    if isinstance(n, str) or n - n != 0 or int(n) != n:  # infinities less themselves are not 0
        raise ValueError(f"{n!r} is no number of tokens")
    return int(n)


class PageBook:
    """Which pages each sequence has, on the host alone: no call here touches a device."""

    def __init__(self, pages: int, page_tokens: int):
        self.pages, self.page_tokens = pages, page_tokens
        self.free_pages = list(range(pages))  # a heap: the lowest first
        self.uses = [0] * pages
        self.sequences = {}  # id -> [length, page numbers]
        self._next = 0

    def _sequence(self, seq):
        if seq not in self.sequences:
            raise KeyError(f"no sequence {seq}")
        return self.sequences[seq]

    def new(self) -> int:
        seq, self._next = self._next, self._next + 1
        self.sequences[seq] = [0, []]
        return seq

    def length(self, seq: int) -> int:
        return self._sequence(seq)[0]

    def used(self) -> int:
        return self.pages - len(self.free_pages)

    def _release(self, page):
        self.uses[page] -= 1
        if self.uses[page] == 0:
            heapq.heappush(self.free_pages, page)

    def _take(self):
        page = heapq.heappop(self.free_pages)
        self.uses[page] = 1
        return page

    def free(self, seq: int):
        for page in self._sequence(seq)[1]:
            self._release(page)
        del self.sequences[seq]

    def fork(self, seq: int) -> int:
        """A sequence with the same tokens, on the same pages."""
        length, pages = self._sequence(seq)
        other = self.new()
        self.sequences[other] = [length, list(pages)]
        for page in pages:
            self.uses[page] += 1
        return other

    def truncate(self, seq: int, length: int):
        """Forgets the tokens from `length` on."""
        s, length = self._sequence(seq), _whole(length)
        if not 0 <= length <= s[0]:
            raise ValueError(f"sequence {seq} has {s[0]} tokens: cannot keep {length}")
        keep = -(-length // self.page_tokens)
        for page in s[1][keep:]:
            self._release(page)
        s[0], s[1] = length, s[1][:keep]

    def grow(self, seqs, counts):
        """Makes room for counts[i] more tokens of seqs[i] and counts them as its own -> (source pages, target pages) to copy
        before the tokens are written: last pages that other sequences share. Raises OutOfPages, and KeyError or ValueError
        for unknown or repeated sequences and negative counts, with nothing changed."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs):
            raise ValueError("seqs must be different sequences, one count for each")
        counts = [_whole(n) for n in counts]
        need, shared = 0, {}
        for seq, n in zip(seqs, counts):
            length, pages = self._sequence(seq)
            if n < 0:
                raise ValueError(f"sequence {seq}: {n} new tokens")
            need += -(-(length + n) // self.page_tokens) - len(pages)
            if n and length % self.page_tokens:  # the last page is written: a copy for all that write it but the last user
                shared.setdefault(pages[-1], []).append(seq)
        for page, writers in shared.items():
            need += min(len(writers), self.uses[page] - 1)
        if need > len(self.free_pages):
            raise OutOfPages(f"{need} pages needed, {len(self.free_pages)} of {self.pages} free")
        src, dst = [], []
        for seq, n in zip(seqs, counts):
            s = self.sequences[seq]
            if n and s[0] % self.page_tokens and self.uses[s[1][-1]] > 1:
                page = self._take()
                src.append(s[1][-1])
                dst.append(page)
                self.uses[s[1][-1]] -= 1
                s[1][-1] = page
            while len(s[1]) * self.page_tokens < s[0] + n:
                s[1].append(self._take())
            s[0] += n
        return src, dst

    def compact(self):
        """Moves the live pages to the lowest numbers -> (source pages, target pages) to copy. No page is both."""
        live = self.used()
        holes = sorted(p for p in self.free_pages if p < live)
        high = [p for p in range(live, self.pages) if self.uses[p]]
        to = dict(zip(high, holes))
        for s in self.sequences.values():
            s[1] = [to.get(p, p) for p in s[1]]
        for a, b in to.items():
            self.uses[b], self.uses[a] = self.uses[a], 0
        self.free_pages = list(range(live, self.pages))
        return list(to.keys()), list(to.values())


@dataclass
class KVStep:
    """The sequences of one forward pass as the kernels read them (int32, on the GPU), and what the host knows of them.
    refresh() of the cache writes a later step of as many sequences into the same tensors, which a captured graph reads."""
    table: torch.Tensor   # [sequences, width] pages, -1 behind a sequence's last
    start: torch.Tensor   # [sequences] tokens before this step
    length: torch.Tensor  # [sequences] tokens with this step's
    cu: torch.Tensor      # [sequences + 1] where each sequence's rows begin
    counts: list
    max_count: int
    max_length: int
    tokens: int           # of all sequences; a call's rows are these, and any padding behind them
    streams: set = field(default_factory=set, repr=False)  # that the allocator knows to read the tensors

    def check(self, rows: torch.Tensor, name: str):
        """The book counts the step's tokens as written: fewer rows than those would leave some of them unwritten."""
        if rows.shape[0] < self.tokens:
            raise ValueError(f"{name} has {rows.shape[0]} rows, the step {self.tokens} tokens")


class _StreamOrder:
    """The order of one cache's work on the GPU: what writes pages comes after all calls before it, what reads them after every
    write before it. Which pages those are the caller cannot see (a fork shares pages until one side writes, a freed page is
    another sequence's next), so the cache itself makes the streams wait for each other where they change; on one stream that is a
    comparison. A wait is for all that the other stream has enqueued by then, replayed graphs too. Streams that made a call
    have to live as long as the cache."""

    def __init__(self, index: int):
        self.index, self.raw, self.writer, self.readers = index, None, None, {}
        if index >= 0:
            self(True)  # the cache's zeros

    def __call__(self, writes: bool, step: KVStep = None):
        if self.index < 0:
            return
        raw = torch._C._cuda_getCurrentRawStream(self.index)
        known = step is None or raw in step.streams
        if known and (raw == self.raw and not self.readers if writes else raw == self.raw or raw in self.readers):
            return
        with torch.cuda.device(self.index):
            if torch.cuda.is_current_stream_capturing():  # this work runs at a replay
                return
        here = torch.cuda.current_stream(self.index)
        if not known:
            for t in (step.table, step.start, step.length, step.cu):
                t.record_stream(here)
            step.streams.add(raw)
        if writes:
            for other in (self.writer, *self.readers.values()):
                if other is not None and other.cuda_stream != raw:
                    here.wait_stream(other)
            self.raw, self.writer, self.readers = raw, here, {}
        elif raw != self.raw and raw not in self.readers:
            if self.writer is not None:
                here.wait_stream(self.writer)
            self.readers[raw] = here


class HBMKVCache:
    """All layers' keys and values on one GPU. dtype: torch.int8, or torch.float8_e4m3fn (values whose magnitudes differ by
    more than int8's 127 steps inside a page)."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, dtype=torch.int8,
                 device="cuda"):
        self.pages = KVPages.empty(layers, pages, kv_heads, head_dim, page_tokens, dtype, device)
        self.device = self.pages.device
        self.book = PageBook(pages, page_tokens)
        self._order = _StreamOrder(self.pages.index)

    def nbytes(self) -> int:
        return self.pages.nbytes()

    # -- sequences ------------------------------------------------------------------------------------------------

    def new(self) -> int:
        return self.book.new()

    def free(self, seq: int):
        self.book.free(seq)

    def fork(self, seq: int) -> int:
        return self.book.fork(seq)

    def truncate(self, seq: int, length: int):
        self.book.truncate(seq, length)

    def length(self, seq: int) -> int:
        return self.book.length(seq)

    def compact(self) -> int:
        """Moves the live pages to the lowest numbers -> how many moved. Steps made before hold pages that are no longer
        theirs: make them anew. Not under capture."""
        self._not_captured()
        self._order(True)
        src, dst = self.book.compact()
        kv_copy(self.pages, src, dst)
        return len(src)

    # -- one forward pass -----------------------------------------------------------------------------------------

    def _not_captured(self):
        """The book counts pages as moved and tokens as there at once: not in a captured graph, which runs later, and often."""
        if self.pages.index >= 0:
            with torch.cuda.device(self.pages.index):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("a cache's step(), refresh() and compact() cannot be captured into a graph")

    @contextlib.contextmanager
    def _given_back(self, seqs, counts):
        """Takes the step's tokens off the book again where its tables are not made, or do not reach the device."""
        try:
            yield
        except BaseException:
            for s, n in zip(seqs, counts):
                self.book.truncate(s, self.book.length(s) - n)
            raise

    def _host_step(self, seqs, counts, width):
        self._not_captured()
        src, dst = self.book.grow(seqs, counts)
        self._order(True)
        kv_copy(self.pages, src, dst)
        with self._given_back(seqs, counts):
            n = len(seqs)
            rows = [self.book.sequences[s] for s in seqs]
            host = np.full((n, width or max([1] + [len(r[1]) for r in rows])), -1, dtype=np.int32)
            for i, r in enumerate(rows):
                host[i, :len(r[1])] = r[1]
            length = np.array([r[0] for r in rows], dtype=np.int32)
            start = length - np.array(counts, dtype=np.int32)
            cu = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
            return host, start, length, cu

    def step(self, seqs, counts, width: int = None) -> KVStep:
        """Room for counts[i] new tokens of sequence seqs[i], which count as its own from here on -> what append and attend
        take. Pages that a fork shares and that are about to be written are copied. width: pages the table has columns for
        (for refresh() of longer sequences; default: as many as the longest has). The tables are uploaded: not under capture.
        The tokens count as written at once: append them on every layer before the sequences are forked, compacted or in another
        step, and where a layer fails take the step back, truncate(seq, length(seq) - count) for each sequence."""
        if not seqs:
            raise ValueError("a step needs a sequence")
        counts = [_whole(c) for c in counts]
        if width is not None:
            self._check_width(seqs, counts, width)
        host, start, length, cu = self._host_step(list(seqs), counts, width)
        with self._given_back(seqs, counts):
            up = [torch.from_numpy(a).to(self.device) for a in (host, start, length, cu)]
        streams = {self._order.raw}  # the one that this was made on
        return KVStep(*up, counts, max(counts), int(length.max()) if width is None else width * self.book.page_tokens, int(cu[-1]),
                      streams)

    def _check_width(self, seqs, counts, width):
        for s, c in zip(seqs, counts):
            if self.book.length(s) + c > width * self.book.page_tokens:
                raise ValueError(f"sequence {s} does not fit {width} pages")

    def refresh(self, step: KVStep, seqs, counts) -> KVStep:
        """A later step of as many sequences with the same counts, written into `step`'s tensors on the current stream: a
        graph that was captured with them then runs this step."""
        counts = [_whole(c) for c in counts]
        if len(seqs) != step.table.shape[0] or counts != step.counts:
            raise ValueError(f"the step was made for {step.table.shape[0]} sequences with counts {step.counts}")
        self._check_width(seqs, counts, step.table.shape[1])
        host, start, length, _ = self._host_step(list(seqs), counts, step.table.shape[1])
        self._order(True, step)
        with self._given_back(seqs, counts):
            for t, a in ((step.table, host), (step.start, start), (step.length, length)):
                t.copy_(torch.from_numpy(a))
        step.max_length = max(step.max_length, int(length.max()))
        return step

    def append(self, layer: int, step: KVStep, k: torch.Tensor, v: torch.Tensor):
        """The step's new keys and values of one layer, bf16 [tokens, kv_heads, head_dim]; kv_append."""
        step.check(k, "k")
        self._order(True, step)
        kv_append(self.pages, layer, k, v, step.table, step.start, step.cu, max_count=step.max_count or 1)

    def attend(self, layer: int, step: KVStep, q: torch.Tensor, scale: float = None, causal: bool = True,
               out: torch.Tensor = None) -> torch.Tensor:
        """The step's rows' attention over one layer of their sequences, bf16 [tokens, heads, head_dim]; kv_attend. Rows of q behind
        the step's tokens (padding) come out as zeros, or stay as they are in `out`."""
        step.check(q, "q")
        if out is None and q.shape[0] > step.tokens:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            out[step.tokens:].zero_()
        self._order(False, step)
        return kv_attend(self.pages, layer, q, step.table, step.length, step.cu, max_count=step.max_count or 1,
                         max_length=step.max_length, scale=scale, causal=causal, out=out)
