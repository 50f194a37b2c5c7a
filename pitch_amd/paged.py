"""Paged caches: the keys and values of many sequences as codes in the pages of one pool, with the operators that a serving
program runs on them (no counterpart in the reference, whose caches are one sequence's contiguous buffers, README.md:65-76).

``PagedCache`` holds (or allocates) a layer's pool. ``PagedAppend`` writes a step's tokens, with the norms of queries and
keys and their position rotation in the same pass; ``PagedDecode`` reads ranges of tokens back; ``PagedAttention`` attends
with one new token of every sequence. Like ``EncodeBatch``, each keeps a call's buffers and checked arguments between
calls, so that ``enqueue()`` costs a few microseconds of host time; the buffers' contents may change between calls, and
``PagedCache.enqueueAppend`` / ``enqueueDecode`` / ``enqueueAttention`` make and issue one such call.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _lib
from .api import (InvalidInput, PITCH, QuantConfig, _buf, _io_type, _lib_or_raise, _raise_for, _stream_handle, _torch)

LAYOUTS = {"head": 0, "token": 1}


def _int(v, name: str, least: int = 0) -> int:
    if isinstance(v, bool) or not isinstance(v, (int, np.integer)) or v < least:
        raise InvalidInput(f"{name} {v!r} must be an integer of at least {least}")
    return int(v)


def _float(v, name: str) -> float:
    try:
        return float(v)
    except (TypeError, ValueError):
        raise InvalidInput(f"{name} {v!r} must be a number") from None


def _device_tensor(t, name: str, dtypes=None):
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise InvalidInput(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise InvalidInput(f"{name} buffer is not device memory")
    if dtypes is not None and t.dtype not in dtypes:
        raise InvalidInput(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    return t


def _vectors(t, name: str, heads: int, dim: int, dtype=None) -> _lib.PitchPagedVectorsC:
    """A [tokens][heads][dim] tensor, strided in its first two dimensions (a slice of a fused projection, a transposed view)."""
    torch = _torch()
    _device_tensor(t, name, None if dtype is None else (dtype,))
    if t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise InvalidInput(f"{name} must be float32, float16 or bfloat16")
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise InvalidInput(f"{name} must be [tokens][{heads}][{dim}], got {list(t.shape)}")
    if t.stride(2) != 1:
        raise InvalidInput(f"{name}: the coordinates of a vector must be neighbours")
    held = t.untyped_storage().nbytes() - t.storage_offset() * t.element_size()
    # the stride of a dimension of one element has no meaning
    ts, hs = (t.stride(i) if t.shape[i] > 1 else t.shape[2] for i in (0, 1))
    return _lib.PitchPagedVectorsC(t.data_ptr(), held, ts, hs)


def _flat(t, name: str, dtype, count: int | None):
    """(pointer, bytes) of a contiguous tensor of this type and number of elements, (None, 0) of None."""
    if t is None:
        return None, 0
    _device_tensor(t, name, (dtype,))
    if count is not None and t.numel() != count:
        raise InvalidInput(f"{name} has {t.numel()} elements; needs {count}")
    return _buf(t, name)


def _tables(t):
    torch = _torch()
    _device_tensor(t, "page tables", (torch.int32,))
    if t.dim() != 2 or t.shape[0] < 1 or t.shape[1] < 1:
        raise InvalidInput(f"page tables must be [sequences][pages], got {list(t.shape)}")
    return _buf(t, "page tables")


class PagedCache:
    """The keys and values of a layer in the pages of a pool: ``pages`` pages of ``pageSize`` token slots (a multiple of 16)
    for each of ``kvHeads`` KV heads, each vector as the codes and the scale that ``enqueueEncode`` writes for ``keyConfig``
    or ``valueConfig`` (default: the same; dimension 64 or 128). ``layout`` "head" puts a page's tokens of a head next to each
    other ([page][head][slot]), "token" a token's heads ([page][slot][head]). Without buffers they are allocated;
    keyCodes / valueCodes are uint8 [page][head][slot][codeStride] (or [page][slot][head][...]), the scales float32 without
    the last dimension. A pool's pages may lie apart (a layer's part of [page][layer][head][slot]): dimension 0 takes any
    stride that is a whole number of vectors, the same for all four buffers."""

    def __init__(self, pitch: PITCH, keyConfig: QuantConfig, valueConfig: QuantConfig | None = None, pages: int = 1,
                 pageSize: int = 64, kvHeads: int = 1, layout: str = "head", keyCodes=None, keyScales=None, valueCodes=None,
                 valueScales=None):
        torch = _torch()
        self.pitch, self.keyConfig, self.valueConfig = pitch, keyConfig, valueConfig or keyConfig
        self.pages, self.pageSize, self.kvHeads = _int(pages, "pages", 1), _int(pageSize, "pageSize", 1), _int(kvHeads, "kvHeads", 1)
        if layout not in LAYOUTS:
            raise InvalidInput(f"layout {layout!r} must be 'head' or 'token'")
        self.layout = layout
        lead = (self.pages,) + ((self.kvHeads, self.pageSize) if layout == "head" else (self.pageSize, self.kvHeads))
        given = [t is not None for t in (keyCodes, keyScales, valueCodes, valueScales)]
        if any(given) and not all(given):
            raise InvalidInput("a cache takes all four buffers or none")
        if not any(given):
            made = []
            for c in (self.keyConfig, self.valueConfig):
                made += [torch.zeros(lead + (c.codeStride,), dtype=torch.uint8, device=pitch.device),
                         torch.zeros(lead, dtype=torch.float32, device=pitch.device)]
            keyCodes, keyScales, valueCodes, valueScales = made
        self.keyCodes, self.keyScales, self.valueCodes, self.valueScales = keyCodes, keyScales, valueCodes, valueScales
        c = _lib.PitchPagedCacheC()
        c.key_config, c.value_config = self.keyConfig._c(), self.valueConfig._c()
        strides = set()
        for name, t, dtype, last in (("key_codes", keyCodes, torch.uint8, self.keyConfig.codeStride),
                                     ("key_scales", keyScales, torch.float32, 1),
                                     ("value_codes", valueCodes, torch.uint8, self.valueConfig.codeStride),
                                     ("value_scales", valueScales, torch.float32, 1)):
            what = name.replace("_", " ")
            _device_tensor(t, what, (dtype,))
            shape = lead + ((last,) if name.endswith("codes") else ())
            if tuple(t.shape) != shape:
                raise InvalidInput(f"{what} must be {list(shape)}, got {list(t.shape)}")
            if not t[0].is_contiguous():
                raise InvalidInput(f"{what}: a page must be contiguous")
            if self.pages > 1:
                if t.stride(0) % last:
                    raise InvalidInput(f"{what}: the pages' stride is no whole number of vectors")
                strides.add(t.stride(0) // last)
            setattr(c, name, t.data_ptr())
            setattr(c, name + "_bytes", t.untyped_storage().nbytes() - t.storage_offset() * t.element_size())
        if len(strides) > 1:
            raise InvalidInput("the four buffers' pages must lie equally far apart")
        c.pages, c.page_size, c.kv_heads, c.layout = self.pages, self.pageSize, self.kvHeads, LAYOUTS[layout]
        c.page_stride = strides.pop() if strides else self.kvHeads * self.pageSize
        self._cstruct = c
        self.attentionWorkspaceBytes(1, 1)   # the library's checks of the pool

    @property
    def dim(self) -> int:
        return self.keyConfig.dim

    def attentionWorkspaceBytes(self, sequences: int, qPerKv: int) -> int:
        """Device workspace that an attention call over this cache needs."""
        call = _lib.PitchPagedAttentionC()
        call.sequences, call.q_per_kv = _int(sequences, "sequences", 1), _int(qPerKv, "qPerKv", 1)
        out = ctypes.c_uint64(0)
        _raise_for(self.pitch._lib.pitch_paged_attention_workspace_size(ctypes.byref(self._cstruct), ctypes.byref(call),
                                                                        ctypes.byref(out)))
        return int(out.value)

    def enqueueAppend(self, keys, values, slots, stream=None, **more) -> None:
        """One PagedAppend call."""
        PagedAppend(self, keys, values, slots, **more).enqueue(stream)

    def enqueueDecode(self, blockTables, rowStarts, stream=None, **more) -> None:
        """One PagedDecode call."""
        PagedDecode(self, blockTables, rowStarts, **more).enqueue(stream)

    def enqueueAttention(self, q, blockTables, lengths, output, stream=None, workspace=None, **more) -> None:
        """One PagedAttention call. On a stream of the caller's, the caller's workspace has to be given: one that is made here
        returns to torch's allocator when the call returns, which orders its next use with the current stream only."""
        if stream is not None and workspace is None:
            raise InvalidInput("a call on a stream of its own needs a workspace of its own")
        PagedAttention(self, q, blockTables, lengths, output, workspace=workspace, **more).enqueue(stream)


class PagedAppend:
    """The write of a step's or a prompt's tokens: keys and values [tokens][kvHeads][dim] are encoded into slots[t] =
    page * pageSize + slot (int64; a token with a slot outside the pool, such as -1 for a batch's padding, is not written).
    Two tokens must not have the same slot. With keyNorm (dim weights of the vectors' type) a key is first divided by
    sqrt(mean(x^2) + eps) and multiplied by the weights; with positions (int64) and the model's tables cos, sin (float32
    [positions][rotaryDim]) its first rotaryDim coordinates are rotated (rotate_half over them). Queries [tokens][heads][dim]
    are normed with queryNorm, rotated and written to queriesOut (the queries themselves, or memory that the call does not
    read; slices of one buffer that share no element are). Tokens with positions
    outside the tables are left out. All vectors have one element type; their first two dimensions take any stride."""

    def __init__(self, cache: PagedCache, keys, values, slots, queries=None, queriesOut=None, queryNorm=None, keyNorm=None,
                 eps: float = 1e-6, cos=None, sin=None, positions=None):
        torch = _torch()
        self.cache = cache
        self._held = (keys, values, slots, queries, queriesOut, queryNorm, keyNorm, cos, sin, positions)
        heads, d = cache.kvHeads, cache.dim
        c = _lib.PitchPagedAppendC()
        c.keys = _vectors(keys, "keys", heads, d)
        c.values = _vectors(values, "values", heads, d, keys.dtype)
        n = keys.shape[0]
        c.io_type, c.tokens = _io_type(keys), n
        if n < 1 or values.shape[0] != n:
            raise InvalidInput(f"keys and values need the same tokens, at least one; got {n} and {values.shape[0]}")
        c.slots, c.slots_bytes = _flat(slots, "slots", torch.int64, n)
        if (queries is None) != (queriesOut is None):
            raise InvalidInput("queries and queriesOut go together")
        if queries is not None:
            if _device_tensor(queries, "queries").dim() != 3 or queries.shape[1] < 1:
                raise InvalidInput(f"queries must be [tokens][heads][dim], got {list(queries.shape)}")
            c.q_heads = queries.shape[1]
            c.queries = _vectors(queries, "queries", c.q_heads, d, keys.dtype)
            c.queries_out = _vectors(queriesOut, "queriesOut", c.q_heads, d, keys.dtype)
            if queries.shape[0] != n or queriesOut.shape[0] != n:
                raise InvalidInput("queries and queriesOut need the keys' tokens")
        c.query_norm, c.query_norm_bytes = _flat(queryNorm, "queryNorm", keys.dtype, d)
        c.key_norm, c.key_norm_bytes = _flat(keyNorm, "keyNorm", keys.dtype, d)
        c.eps = _float(eps, "eps")
        if positions is not None:
            if cos is None or sin is None:
                raise InvalidInput("positions need tables cos and sin [positions][rotaryDim]")
            if _device_tensor(cos, "cos").dim() != 2 or cos.shape != _device_tensor(sin, "sin").shape or cos.shape[0] < 1:
                raise InvalidInput("cos and sin must be [positions][rotaryDim], both the same")
            c.positions, c.positions_bytes = _flat(positions, "positions", torch.int64, n)
            c.cos, c.table_bytes = _flat(cos, "cos", torch.float32, None)
            c.sin, _ = _flat(sin, "sin", torch.float32, None)
            c.rotary_dim = cos.shape[1]
        elif cos is not None or sin is not None:
            raise InvalidInput("cos and sin need positions")
        self._call, self._ref, self._pool = c, ctypes.byref(c), ctypes.byref(cache._cstruct)
        self._fn, self._device = cache.pitch._lib.pitch_enqueue_paged_append, cache.pitch.device

    def enqueue(self, stream=None) -> None:
        rc = self._fn(self._pool, self._ref, _stream_handle(stream, self._device))
        if rc:
            _raise_for(rc)


class PagedDecode:
    """Reads tokens back: row r of keysOut / valuesOut [rows][kvHeads][dim] (one may be left out) with rowStarts[b] <= r <
    rowStarts[b + 1] (int32, sequences + 1 of them, not decreasing) is token firstTokens[b] (int32, default 0) + r -
    rowStarts[b] of sequence b, whose page is blockTables[b][token // pageSize] (int32). Other rows, and rows whose page lies
    outside the pool or the table, are left as they were. The outputs' token strides are at most 2^22 elements; the two may be
    slices of one buffer that share no element."""

    def __init__(self, cache: PagedCache, blockTables, rowStarts, keysOut=None, valuesOut=None, firstTokens=None):
        torch = _torch()
        self.cache = cache
        self._held = (blockTables, rowStarts, keysOut, valuesOut, firstTokens)
        outs = [t for t in (keysOut, valuesOut) if t is not None]
        if not outs:
            raise InvalidInput("keysOut or valuesOut is needed")
        c = _lib.PitchPagedDecodeC()
        if keysOut is not None:
            c.keys = _vectors(keysOut, "keysOut", cache.kvHeads, cache.dim)
        if valuesOut is not None:
            c.values = _vectors(valuesOut, "valuesOut", cache.kvHeads, cache.dim, outs[0].dtype)
        c.io_type, c.rows = _io_type(outs[0]), outs[0].shape[0]
        if c.rows < 1 or outs[-1].shape[0] != c.rows:
            raise InvalidInput("keysOut and valuesOut need the same rows, at least one")
        c.block_tables, c.block_tables_bytes = _tables(blockTables)
        c.sequences, c.table_width = blockTables.shape
        c.row_starts, c.row_starts_bytes = _flat(rowStarts, "rowStarts", torch.int32, c.sequences + 1)
        c.first_tokens, c.first_tokens_bytes = _flat(firstTokens, "firstTokens", torch.int32, c.sequences)
        self._call, self._ref, self._pool = c, ctypes.byref(c), ctypes.byref(cache._cstruct)
        self._fn, self._device = cache.pitch._lib.pitch_enqueue_paged_decode, cache.pitch.device

    def enqueue(self, stream=None) -> None:
        rc = self._fn(self._pool, self._ref, _stream_handle(stream, self._device))
        if rc:
            _raise_for(rc)


class PagedAttention:
    """One new token of every sequence over its pages: q and output [sequences][heads][dim] float16 or bfloat16 (heads =
    kvHeads * 1..8; strided as in PagedAppend; at most 2,048 sequences; the output may be q itself), blockTables int32 [sequences][pages], lengths
    int32 [sequences] with the new token counted. The scores are softcap * tanh(scale q.k / softcap) (softcap 0: scale q.k; scale defaults to 1 / sqrt(dim))
    plus slopes[h] * (t - (length - 1)) (float32 [heads]) over the last ``window`` tokens (0: all). lse, float32
    [sequences][heads], receives the natural-log sum of exp. A sequence of length 0 gives zeros (and minus infinity). Without
    a workspace one is allocated and held, and a call on another stream waits for the work of the stream that it was allocated on;
    a graph needs the object as long as it is replayed. Two calls that may run at the same time must not share a workspace."""

    def __init__(self, cache: PagedCache, q, blockTables, lengths, output, scale: float | None = None, softcap: float = 0.0,
                 window: int = 0, slopes=None, lse=None, workspace=None):
        torch = _torch()
        self.cache = cache
        c = _lib.PitchPagedAttentionC()
        _device_tensor(q, "q", (torch.float16, torch.bfloat16))
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % cache.kvHeads:
            raise InvalidInput(f"q must be [sequences][a multiple of {cache.kvHeads} heads][{cache.dim}], got {list(q.shape)}")
        heads = q.shape[1]
        c.queries = _vectors(q, "q", heads, cache.dim)
        c.output = _vectors(output, "output", heads, cache.dim, q.dtype)
        c.io_type, c.sequences, c.q_per_kv, c.window = _io_type(q), q.shape[0], heads // cache.kvHeads, _int(window, "window")
        c.block_tables, c.block_tables_bytes = _tables(blockTables)
        if output.shape[0] != c.sequences or blockTables.shape[0] != c.sequences:
            raise InvalidInput("q, output and blockTables need the same sequences")
        c.table_width = blockTables.shape[1]
        c.lengths, c.lengths_bytes = _flat(lengths, "lengths", torch.int32, c.sequences)
        c.slopes, c.slopes_bytes = _flat(slopes, "slopes", torch.float32, heads)
        c.lse, c.lse_bytes = _flat(lse, "lse", torch.float32, c.sequences * heads)
        c.scale = 1.0 / math.sqrt(cache.dim) if scale is None else _float(scale, "scale")
        c.softcap = _float(softcap, "softcap")
        # the handles of the streams that may use the workspace as it is (None: all, the caller's workspace is the caller's to order)
        self._own, self._ready = None, None
        if workspace is None:
            n = cache.attentionWorkspaceBytes(c.sequences, c.q_per_kv)
            if n:
                workspace = torch.empty(n, dtype=torch.uint8, device=cache.pitch.device)
                self._own = torch.cuda.current_stream(cache.pitch.device)
                self._ready = {self._own.cuda_stream}
        if workspace is not None:
            c.workspace, c.workspace_bytes = _buf(workspace, "workspace")
        self._held = (q, blockTables, lengths, output, slopes, lse, workspace)
        self._call, self._ref, self._pool = c, ctypes.byref(c), ctypes.byref(cache._cstruct)
        self._fn, self._device = cache.pitch._lib.pitch_enqueue_paged_attention, cache.pitch.device

    def enqueue(self, stream=None) -> None:
        handle = _stream_handle(stream, self._device)
        if self._ready is not None and handle not in self._ready:
            self._admit(stream, handle)
        rc = self._fn(self._pool, self._ref, handle)
        if rc:
            _raise_for(rc)

    def _admit(self, stream, handle: int) -> None:
        """Lets another stream use a workspace allocated here: behind the work that the allocation's stream holds (the memory may
        have been freed by it just before), and known to torch's allocator, which else hands it out again on its own stream
        as soon as this object is gone."""
        torch = _torch()
        if stream is None:
            stream = torch.cuda.current_stream(self._device)
        elif not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(handle, device=self._device) if handle else torch.cuda.default_stream(self._device)
        self._held[-1].record_stream(stream)
        with torch.cuda.stream(stream):
            capturing = torch.cuda.is_current_stream_capturing()
        if not capturing:   # (a graph cannot wait for work outside of it; torch.cuda.graph begins with a synchronisation)
            stream.wait_event(self._own.record_event())
            self._ready.add(handle)
