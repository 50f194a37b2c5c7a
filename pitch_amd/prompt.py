"""Attention over whole prompts (no counterpart in the reference, whose next step is attention, README.md:96): packed sequences of
queries over their keys and values, causal with grouped heads. It stands between ``PagedAppend``, which writes a prompt's tokens to the
cache, and ``PagedAttention``, which attends with one new token; a chunk behind a prefix takes the rows that ``PagedDecode`` reads back.
"""
from __future__ import annotations

import ctypes
import math

from . import _lib
from .api import InvalidInput, PITCH, _io_type, _raise_for, _torch
from .paged import WorkspaceCall, _device_tensor, _flat, _float, _int, _vectors


class PromptAttention(WorkspaceCall):
    """q and output [rows][heads][dim], k and v [keys][kvHeads][dim], float16 or bfloat16, dim 64 or 128, heads a multiple of kvHeads;
    the first two dimensions take any strides that are multiples of 16 bytes (slices of a fused projection), k and v token strides of
    up to 2^22 elements. Sequence b has the rows rowStarts[b] <= r < rowStarts[b + 1] (int32, sequences + 1 of them, not
    decreasing) and the keys keyStarts[b] <= r < keyStarts[b + 1] (default: the same rows); its queries are the last of its tokens,
    query i of nq at position p = nk - nq + i. A query sees its sequence's keys, with ``causal`` up to its own position, with a
    ``window`` the last ``window`` of these (0: all). The scores are softcap * tanh(scale q.k / softcap) (softcap 0: scale q.k; scale
    defaults to 1 / sqrt(dim)) plus slopes[h] * (j - p) (float32 [heads]). Window and slopes need ``causal``. lse, float32
    [rows][heads], receives the natural-log sum of exp. A query that sees no key gives zeros (and minus infinity); rows of no sequence
    are left as they were; the output may be q itself. Like ``PagedAttention``, the object keeps the checked arguments and, without a
    workspace of the caller's, one that is allocated here (few queries over long keys need one): two calls that may run at the same time
    must not share it (the program orders one object's calls on several streams), and a graph needs the object as long as it is
    replayed. ``workspaceBytes`` is 0, or on 256 compute units up to 136 MB for heads of 128 and 69 MB for heads of 64, few queries or many:
    the layers of a step, whose calls follow each other on one stream, are best given one ``workspace`` (uint8) of that size."""

    def __init__(self, pitch: PITCH, q, k, v, rowStarts, output, keyStarts=None, causal: bool = True, scale: float | None = None,
                 softcap: float = 0.0, window: int = 0, slopes=None, lse=None, workspace=None):
        torch = _torch()
        c = _lib.PitchPromptAttentionC()
        for name, t in (("q", q), ("k", k)):
            if _device_tensor(t, name, (torch.float16, torch.bfloat16)).dim() != 3 or 0 in t.shape:
                raise InvalidInput(f"{name} must be [tokens][heads][dim], got {list(t.shape)}")
        heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
        if heads % kv:
            raise InvalidInput(f"the query heads ({heads}) must be a multiple of the KV heads ({kv})")
        if not isinstance(causal, bool):
            raise InvalidInput(f"causal {causal!r} must be True or False")
        c.queries, c.keys = _vectors(q, "q", heads, dim), _vectors(k, "k", kv, dim, q.dtype)
        c.values, c.output = _vectors(v, "v", kv, dim, q.dtype), _vectors(output, "output", heads, dim, q.dtype)
        if v.shape[0] != k.shape[0] or output.shape[0] != q.shape[0]:
            raise InvalidInput("k and v, and q and output, need the same tokens")
        if _device_tensor(rowStarts, "rowStarts").dim() != 1 or rowStarts.shape[0] < 2:
            raise InvalidInput(f"rowStarts must be [sequences + 1], got {list(rowStarts.shape)}")
        starts = rowStarts.shape[0]
        c.row_starts, c.row_starts_bytes = _flat(rowStarts, "rowStarts", torch.int32, starts)
        if keyStarts is None:
            keyStarts = rowStarts
        c.key_starts, c.key_starts_bytes = _flat(keyStarts, "keyStarts", torch.int32, starts)
        c.slopes, c.slopes_bytes = _flat(slopes, "slopes", torch.float32, heads)
        c.lse, c.lse_bytes = _flat(lse, "lse", torch.float32, q.shape[0] * heads)
        c.io_type, c.dim, c.sequences, c.q_heads, c.kv_heads = _io_type(q), dim, starts - 1, heads, kv
        c.causal, c.window, c.rows, c.key_rows = causal, _int(window, "window"), q.shape[0], k.shape[0]
        if c.window != window:
            raise InvalidInput(f"window {window} must be below 2^31")
        c.scale = 1.0 / math.sqrt(dim) if scale is None else _float(scale, "scale")
        c.softcap = _float(softcap, "softcap")
        needed = ctypes.c_uint64(0)
        _raise_for(pitch._lib.pitch_prompt_attention_workspace_size(ctypes.byref(c), ctypes.byref(needed)))
        self.workspaceBytes = int(needed.value)   # device workspace that the call needs
        self._hold_workspace(c, workspace, self.workspaceBytes, pitch.device)
        self._held = (q, k, v, rowStarts, output, keyStarts, slopes, lse)
        self._call, self._ref = c, ctypes.byref(c)
        self._fn, self._device = pitch._lib.pitch_enqueue_prompt_attention, pitch.device

    def enqueue(self, stream=None) -> None:
        rc = self._fn(self._ref, self._handle(stream))
        if rc:
            _raise_for(rc)
