"""Page tables in device memory (no counterpart in the reference, whose caches are one sequence's contiguous buffers,
README.md:65-76): ``PagedTables`` holds (or allocates) the tables, lengths and counts of references of sequences whose layers'
``PagedCache`` pools have the same pages. ``PagedReserve`` hands out pages and slots for new tokens, ``PagedTrim`` gives tokens back,
``PagedFork`` makes rows copies of others, sharing whole pages, and ``PagedCompact`` moves the pages in use to the lowest numbers. Nothing
is read back to the host, so a captured graph serves every step: reserve, append, attend. Like ``PagedAttention``, each keeps a
call's checked arguments between calls; ``PagedTables.enqueueReserve`` and the like make and issue one such call.
"""
from __future__ import annotations

import ctypes
import threading

from . import _lib
from .api import InvalidInput, _raise_for, _torch
from .paged import PagedCache, WorkspaceCall, _device_tensor, _flat, _int, _tables


class PagedTables(WorkspaceCall):
    """The pages of sequences over the pools of ``caches`` (the layers' PagedCache objects, or one; all with as many pages of the same
    size): sequence b holds blockTables[b][0 .. ceil(lengths[b] / pageSize) - 1]. blockTables int32 [sequences][width], lengths int32
    [sequences], references int32 [pages] (how many entries hold a page; free where not positive) and missing int32 [1] (pages that the
    last reserve or fork lacked) are allocated empty, for ``sequences`` rows (at most 2,048) of ``width`` pages, or given. A
    program that keeps a page for itself, a prefix's say, adds 1 to its references. Free pages are handed out lowest
    number first, in the order of the sequences and their tokens. Where they run out, a row ends with its last token that has a
    page. Calls on the same tables run one after the other, in the order in which they are made: on another stream than the last one's, or
    the first on another than the one that the tables were made on, a call waits for that stream's work. (A captured call waits for
    nothing outside of its graph, and nothing waits for it: the program orders captured calls of several streams, and replays. So it does
    appends to the pools and attention over them.)"""

    def __init__(self, caches, sequences: int | None = None, width: int | None = None, blockTables=None, lengths=None, references=None,
                 missing=None):
        torch = _torch()
        self.caches = [caches] if isinstance(caches, PagedCache) else list(caches) if isinstance(caches, (list, tuple)) else []
        if not self.caches or not all(isinstance(c, PagedCache) for c in self.caches):
            raise InvalidInput("caches must be PagedCache objects, at least one")
        first = self.caches[0]
        self.pitch, self.pages, self.pageSize = first.pitch, first.pages, first.pageSize
        if any((c.pages, c.pageSize) != (self.pages, self.pageSize) for c in self.caches):
            raise InvalidInput("all caches need as many pages of the same size")
        device, given = self.pitch.device, blockTables is not None
        if blockTables is None:
            if sequences is None or width is None:
                raise InvalidInput("sequences and width are needed where blockTables is not given")
            blockTables = torch.full((_int(sequences, "sequences", 1), _int(width, "width", 1)), -1, dtype=torch.int32, device=device)
        elif sequences is not None or width is not None:
            raise InvalidInput("blockTables has its own sequences and width")
        c = _lib.PitchPagedTablesC()
        c.block_tables, c.block_tables_bytes = _tables(blockTables)
        self.sequences, self.width = blockTables.shape
        made = [] if given else [blockTables]   # what is allocated here, as the workspace is

        def zeros(n):
            made.append(torch.zeros(n, dtype=torch.int32, device=device))
            return made[-1]

        lengths = zeros(self.sequences) if lengths is None else lengths
        references = zeros(self.pages) if references is None else references
        missing = zeros(1) if missing is None else missing
        c.lengths, c.lengths_bytes = _flat(lengths, "lengths", torch.int32, self.sequences)
        c.references, c.references_bytes = _flat(references, "references", torch.int32, self.pages)
        c.missing, c.missing_bytes = _flat(missing, "missing", torch.int32, 1)
        c.table_width, c.pages, c.page_size, c.sequences = self.width, self.pages, self.pageSize, self.sequences
        self.blockTables, self.lengths, self.references, self.missing = blockTables, lengths, references, missing
        needed = ctypes.c_uint64(0)
        _raise_for(self.pitch._lib.pitch_paged_tables_workspace_size(ctypes.byref(c), ctypes.byref(needed)))
        self._hold_workspace(c, None, int(needed.value), device)
        self._made = made
        self._cstruct, self._device = c, device
        # the stream of the last call, or an event behind it, and the stream's handle where a call on it needs no wait
        self._last, self._last_handle, self._turn = self._own, self._own.cuda_stream, threading.Lock()
        self._layers = (_lib.PitchPagedCacheC * len(self.caches))(*[cache._cstruct for cache in self.caches])

    def enqueueReserve(self, newTokens, slots, positions=None, stream=None) -> None:
        """One PagedReserve call."""
        PagedReserve(self, newTokens, slots, positions=positions).enqueue(stream)

    def enqueueTrim(self, keep, stream=None) -> None:
        """One PagedTrim call."""
        PagedTrim(self, keep).enqueue(stream)

    def enqueueFork(self, parents, stream=None) -> None:
        """One PagedFork call."""
        PagedFork(self, parents).enqueue(stream)

    def enqueueCompact(self, mapping=None, used=None, stream=None) -> None:
        """One PagedCompact call."""
        PagedCompact(self, mapping=mapping, used=used).enqueue(stream)

    def _admit(self, stream, handle: int) -> None:
        super()._admit(stream, handle)
        for t in self._made:
            t.record_stream(self._stream(stream, handle))

    def _capturing(self, stream) -> bool:
        torch = _torch()
        with torch.cuda.stream(stream):
            return torch.cuda.is_current_stream_capturing()

    def _issue(self, launch, stream) -> int:
        """Makes a call behind the last one on these tables."""
        with self._turn:   # (two threads' calls: the second looks for the first when that has been made)
            handle = self._handle(stream)
            if handle == self._last_handle:
                return launch(handle)
            now = self._stream(stream, handle)
            if self._capturing(now):
                return launch(handle)
            if isinstance(self._last, _torch().cuda.Event):
                now.wait_event(self._last)
            elif not self._capturing(self._last):   # (a capture that has begun since then began behind all of the device's work)
                now.wait_event(self._last.record_event())
            rc = launch(handle)
            # A stream that is not torch's own, known by a number that is its handle, may be gone before the next call, or another one with
            # the same handle in its place: its event is recorded now. Torch's own streams stay, and cost their calls nothing.
            if handle and now.stream_id == handle:
                self._last, self._last_handle = now.record_event(), None
            else:
                self._last, self._last_handle = now, handle
            return rc


class _TablesCall:
    """A call on tables, whose workspace is the tables'."""

    def __init__(self, tables: PagedTables):
        if not isinstance(tables, PagedTables):
            raise InvalidInput("tables must be a PagedTables object")
        self.tables = tables
        self._pool, self._lib = ctypes.byref(tables._cstruct), tables.pitch._lib

    def enqueue(self, stream=None) -> None:
        rc = self.tables._issue(self._launch, stream)
        if rc:
            _raise_for(rc)


class PagedReserve(_TablesCall):
    """Takes newTokens[b] (int32 [sequences]; 0 or less: none) further tokens into every sequence b: hands out pages where those that
    it holds do not suffice, and adds to lengths. The tokens are packed in the order of the sequences; token t's slot (page * pageSize +
    slot, for ``PagedAppend``) goes to slots[t] and its position in its sequence to positions[t] (int64, both as many as a step has
    room for). A token without a page, or without a place in its row of the table, has -1 in both, and so have the entries behind the last
    token: ``PagedAppend`` leaves them out. Tokens for which slots has no room are not taken."""

    def __init__(self, tables: PagedTables, newTokens, slots, positions=None):
        super().__init__(tables)
        torch = _torch()
        c = _lib.PitchPagedReserveC()
        c.new_tokens, c.new_tokens_bytes = _flat(newTokens, "newTokens", torch.int32, tables.sequences)
        c.capacity = _device_tensor(slots, "slots", (torch.int64,)).numel()
        c.slots, c.slots_bytes = _flat(slots, "slots", torch.int64, None)
        c.positions, c.positions_bytes = _flat(positions, "positions", torch.int64, c.capacity)
        self._held, self._call, self._ref = (newTokens, slots, positions), c, ctypes.byref(c)

    def _launch(self, handle: int) -> int:
        return self._lib.pitch_enqueue_paged_reserve(self._pool, self._ref, handle)


class PagedTrim(_TablesCall):
    """Cuts every sequence b to at most keep[b] tokens (int32 [sequences]; 0 or less: the whole sequence is given back). The pages
    behind lose a reference; what remains is untouched.

    A row that is cut below the length that it had in the last fork, as parent or as child, may end within a page that another row holds as well. It shares
    that page from then on partly filled, and PagedReserve, which looks at lengths and not at who else holds a page, would have its next
    tokens written over the other's. (Rows that are cut by no more than they have grown since, drafted tokens, are not concerned.) Such a row
    is forked into an empty one, which gets that page as a copy, and given back behind that. A program that cannot know which rows these
    are, a captured step, gives its n rows n empty ones and forks with the parents 0 .. n - 1, 0 .. n - 1, then n .. 2 n - 1 and n
    times -1: behind that every row is what it was, and its partly filled last page its own. It takes a free page and a copy of that page's
    tokens for each row that ends within a page; with ``missing`` above 0 behind the first of the two, rows have lost their last tokens."""

    def __init__(self, tables: PagedTables, keep):
        super().__init__(tables)
        self._held, (self._keep, self._bytes) = keep, _flat(keep, "keep", _torch().int32, tables.sequences)

    def _launch(self, handle: int) -> int:
        return self._lib.pitch_enqueue_paged_trim(self._pool, self._keep, self._bytes, handle)


class PagedFork(_TablesCall):
    """Makes every row b a copy of row parents[b] (int32 [sequences]) as it was before the call; b itself leaves the row alone, a number
    outside the rows (-1) empties it. Whole pages are shared; a partly filled last page goes to one row (the parent's own if that stays,
    else its first child), and the others get a page of their own with its tokens, in every cache of the tables."""

    def __init__(self, tables: PagedTables, parents):
        super().__init__(tables)
        self._held, (self._parents, self._bytes) = parents, _flat(parents, "parents", _torch().int32, tables.sequences)

    def _launch(self, handle: int) -> int:
        t = self.tables
        return self._lib.pitch_enqueue_paged_fork(self._pool, t._layers, len(t.caches), self._parents, self._bytes, handle)


class PagedCompact(_TablesCall):
    """Moves the pages in use to the lowest numbers: with U in use, those at U and above go into the free ones below U, the k-th to the
    k-th, in every cache; tables and references follow. mapping (int32 [pages]) receives each page's new number, -1 for a free
    page, and used (int32 [1]) U."""

    def __init__(self, tables: PagedTables, mapping=None, used=None):
        super().__init__(tables)
        torch = _torch()
        self._held = (mapping, used)
        self._more = _flat(mapping, "mapping", torch.int32, tables.pages) + _flat(used, "used", torch.int32, 1)

    def _launch(self, handle: int) -> int:
        t = self.tables
        return self._lib.pitch_enqueue_paged_compact(self._pool, t._layers, len(t.caches), *self._more, handle)
