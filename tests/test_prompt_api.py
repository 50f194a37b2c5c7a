"""Prompt attention's and the page tables' entry points without a GPU: every argument that can be checked on the host is, before the
library looks for a device. The buffers are host memory and never reach a kernel."""
import ctypes

import pytest

from pitch_amd import _lib
from test_paged_api import DIM, HEADS, PAGE, PAGES, Memory, _cache, lib  # noqa: F401 (lib: a fixture)

B, ROWS, KEYS, Q, WIDTH = 3, 40, 60, 4, 6
BAD, DIMENSION, MISMATCH = _lib.ERR_INVALID_INPUT, _lib.ERR_INVALID_DIMENSION, _lib.ERR_CONFIGURATION_MISMATCH


def _stopped_at_the_device(lib, rc):  # noqa: F811
    return rc == _lib.ERR_DEVICE_UNAVAILABLE or (rc == BAD and "not device memory" in lib.pitch_last_error().decode())


def _vectors(mem, tokens, heads):
    nbytes = tokens * heads * DIM * 2
    return _lib.PitchPagedVectorsC(mem(nbytes), nbytes, heads * DIM, DIM)


def _prompt(mem):
    c = _lib.PitchPromptAttentionC()
    c.io_type, c.dim, c.sequences, c.q_heads, c.kv_heads, c.causal, c.rows, c.key_rows = _lib.IO_BF16, DIM, B, Q, HEADS, 1, ROWS, KEYS
    c.queries, c.output = _vectors(mem, ROWS, Q), _vectors(mem, ROWS, Q)
    c.keys, c.values = _vectors(mem, KEYS, HEADS), _vectors(mem, KEYS, HEADS)
    for name, size in (("row_starts", 4 * (B + 1)), ("key_starts", 4 * (B + 1)), ("slopes", 4 * Q), ("lse", 4 * Q * ROWS)):
        setattr(c, name, mem(size))
        setattr(c, name + "_bytes", size)
    c.scale, c.workspace, c.workspace_bytes = 0.1, mem(1 << 16), 1 << 40
    return c


def _issue(lib, change=lambda c, mem: None):  # noqa: F811
    mem = Memory()
    c = _prompt(mem)
    change(c, mem)
    return lib.pitch_enqueue_prompt_attention(ctypes.byref(c), None)


def _set(**fields):
    def change(c, mem):
        for name, v in fields.items():
            setattr(c, name, v)
    return change


def _vec(which, **fields):
    def change(c, mem):
        for name, v in fields.items():
            setattr(getattr(c, which), name, v(getattr(getattr(c, which), name)) if callable(v) else v)
    return change


def test_a_prompt_without_a_fault_stops_at_the_device(lib):  # noqa: F811
    assert _stopped_at_the_device(lib, _issue(lib))
    assert _stopped_at_the_device(lib, _issue(lib, _set(slopes=None, lse=None, causal=0)))
    assert _stopped_at_the_device(lib, _issue(lib, _set(softcap=5.0, window=2 ** 31 - 1, scale=-1.0)))


@pytest.mark.parametrize("change,code", [
    (_set(io_type=0), BAD), (_set(io_type=3), BAD), (_set(dim=32), DIMENSION), (_set(dim=96), DIMENSION), (_set(sequences=0), BAD),
    (_set(sequences=1 << 24), BAD), (_set(q_heads=0), BAD), (_set(kv_heads=0), BAD), (_set(q_heads=3), BAD), (_set(causal=2), BAD),
    (_set(reserved=1), BAD), (_set(window=2 ** 31), BAD), (_set(causal=0, window=4, slopes=None), BAD), (_set(causal=0), BAD), (_set(rows=0), BAD),
    (_set(rows=ROWS + 1), BAD), (_set(rows=2 ** 30), BAD), (_set(key_rows=0), BAD), (_set(key_rows=KEYS + 1), BAD), (_set(key_rows=2 ** 31), BAD),
    (_set(row_starts=None), BAD), (_set(row_starts_bytes=4 * B), BAD), (_set(key_starts=None), BAD), (_set(key_starts_bytes=4 * B), BAD),
    (_set(slopes_bytes=4 * Q - 4), BAD), (_set(lse_bytes=4 * Q * ROWS - 4), BAD), (_set(scale=float("nan")), BAD),
    (_set(scale=float("inf")), BAD), (_set(softcap=-1.0), BAD), (_set(softcap=float("nan")), BAD),
    (_vec("queries", data=None), BAD), (_vec("queries", data=lambda p: p + 8), BAD), (_vec("keys", token_stride=HEADS * DIM + 4), BAD),
    (_vec("values", head_stride=DIM + 2), BAD), (_vec("output", bytes=lambda n: n - 2), BAD), (_vec("output", token_stride=DIM), BAD),
    (_vec("output", head_stride=0), BAD), (_vec("keys", token_stride=(1 << 22) + 8, bytes=1 << 60), BAD)])
def test_prompt_refusals(lib, change, code):  # noqa: F811
    assert _issue(lib, change) == code
    assert "device" not in lib.pitch_last_error().decode()


@pytest.mark.parametrize("out", ["output", "lse"])
@pytest.mark.parametrize("name", ["queries", "keys", "values", "row_starts", "key_starts", "slopes"])
def test_prompt_outputs_that_overlap_inputs(lib, out, name):  # noqa: F811
    def change(c, mem):
        at = getattr(c, name)
        at = at.data if isinstance(at, _lib.PitchPagedVectorsC) else at
        room = mem(1 << 16)
        if out == "lse":
            c.lse = at if name in ("queries", "keys", "values") else room
        else:
            c.output.data = room if name not in ("queries", "keys", "values") else at + (256 if name == "queries" else 0)
            c.output.bytes = 1 << 40
        if name in ("row_starts", "key_starts", "slopes"):
            setattr(c, name, room + 16)
    assert _issue(lib, change) == BAD and "overlap" in lib.pitch_last_error().decode()


def test_a_prompt_in_place_is_taken(lib):  # noqa: F811
    assert _stopped_at_the_device(lib, _issue(lib, lambda c, mem: setattr(c.output, "data", c.queries.data)))


def _tables(mem):
    t = _lib.PitchPagedTablesC()
    t.table_width, t.pages, t.page_size, t.sequences = WIDTH, PAGES, PAGE, B
    need = ctypes.c_uint64(0)
    assert _lib.load().pitch_paged_tables_workspace_size(ctypes.byref(t), ctypes.byref(need)) == 0 and need.value > 0
    for name, size in (("block_tables", 4 * WIDTH * B), ("lengths", 4 * B), ("references", 4 * PAGES), ("missing", 4), ("workspace", need.value)):
        setattr(t, name, mem(size))
        setattr(t, name + "_bytes", size)
    return t


def _reserve(mem):
    c = _lib.PitchPagedReserveC()
    c.capacity = 9
    for name, size in (("new_tokens", 4 * B), ("slots", 72), ("positions", 72)):
        setattr(c, name, mem(size))
        setattr(c, name + "_bytes", size)
    return c


def _calls(lib, mem, t, caches, n=1):  # noqa: F811
    """Every call on the tables, by name."""
    r, ref = _reserve(mem), ctypes.byref(t)
    rows = mem(4 * B)
    return {"reserve": lambda: lib.pitch_enqueue_paged_reserve(ref, ctypes.byref(r), None),
            "trim": lambda: lib.pitch_enqueue_paged_trim(ref, rows, 4 * B, None),
            "fork": lambda: lib.pitch_enqueue_paged_fork(ref, caches, n, rows, 4 * B, None),
            "compact": lambda: lib.pitch_enqueue_paged_compact(ref, caches, n, mem(4 * PAGES), 4 * PAGES, mem(4), 4, None)}


CALLS = ["reserve", "trim", "fork", "compact"]


def _tables_call(lib, name, change=lambda t, mem: None, cache=lambda c, mem: None, n=1):  # noqa: F811
    mem = Memory()
    t, c = _tables(mem), (_lib.PitchPagedCacheC * 1)(_cache(lib, mem))
    change(t, mem)
    cache(c[0], mem)
    return _calls(lib, mem, t, c, n)[name]()


@pytest.mark.parametrize("name", CALLS)
def test_tables_without_a_fault_stop_at_the_device(lib, name):  # noqa: F811
    assert _stopped_at_the_device(lib, _tables_call(lib, name))
    assert _stopped_at_the_device(lib, _tables_call(lib, name, _set(missing=None, missing_bytes=0)))


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("change", [
    _set(table_width=0), _set(table_width=WIDTH + 1), _set(table_width=2 ** 27), _set(pages=0), _set(pages=PAGES + 1), _set(pages=2 ** 28),
    _set(page_size=0), _set(page_size=24), _set(page_size=2 ** 17), _set(sequences=0), _set(sequences=B + 1), _set(sequences=2049),
    _set(block_tables=None), _set(block_tables_bytes=4), _set(lengths=None), _set(lengths_bytes=4), _set(references=None),
    _set(references_bytes=4 * PAGES - 4), _set(missing_bytes=3), _set(workspace=None), _set(workspace_bytes=64),
    lambda t, mem: setattr(t, "workspace", t.workspace + 4), lambda t, mem: setattr(t, "lengths", t.lengths + 2),
    lambda t, mem: setattr(t, "lengths", t.block_tables + 8), lambda t, mem: setattr(t, "missing", t.references),
    lambda t, mem: setattr(t, "references", t.workspace + 64)])
def test_tables_refusals(lib, name, change):  # noqa: F811
    assert _tables_call(lib, name, change) == BAD
    assert "device" not in lib.pitch_last_error().decode()


@pytest.mark.parametrize("change", [
    _set(capacity=0), _set(capacity=10), _set(capacity=2 ** 31), _set(new_tokens=None), _set(new_tokens_bytes=4), _set(slots=None),
    _set(slots_bytes=64), _set(positions_bytes=64), lambda c, mem: setattr(c, "slots", c.slots + 4),
    lambda c, mem: setattr(c, "positions", c.slots + 64), lambda c, mem: setattr(c, "new_tokens", c.slots + 8)])
def test_reserve_refusals(lib, change):  # noqa: F811
    mem = Memory()
    t, c = _tables(mem), _reserve(mem)
    change(c, mem)
    assert lib.pitch_enqueue_paged_reserve(ctypes.byref(t), ctypes.byref(c), None) == BAD
    assert "device" not in lib.pitch_last_error().decode()


@pytest.mark.parametrize("name", ["fork", "compact"])
def test_refusals_of_caches(lib, name):  # noqa: F811
    assert _tables_call(lib, name, n=0) == BAD
    assert _tables_call(lib, name, n=5000) == BAD
    assert _tables_call(lib, name, cache=_set(key_codes=None)) == BAD
    assert _tables_call(lib, name, cache=_set(value_scales_bytes=4)) == BAD
    assert _tables_call(lib, name, cache=_set(pages=PAGES - 1)) == MISMATCH
    assert _tables_call(lib, name, cache=_set(page_size=16)) == MISMATCH
    # tables inside of a pool
    assert _tables_call(lib, name, cache=lambda c, mem: setattr(c, "key_scales", c.key_codes), change=lambda t, mem: None) in (BAD, _lib.ERR_DEVICE_UNAVAILABLE)
    mem = Memory()
    t, c = _tables(mem), (_lib.PitchPagedCacheC * 1)(_cache(lib, mem))
    t.lengths = c[0].value_codes + 128
    assert _calls(lib, mem, t, c)[name]() == BAD and "overlap" in lib.pitch_last_error().decode()


@pytest.mark.parametrize("name", ["trim", "fork", "compact"])
def test_refusals_of_rows(lib, name):  # noqa: F811
    mem = Memory()
    t, c = _tables(mem), (_lib.PitchPagedCacheC * 1)(_cache(lib, mem))
    ref = ctypes.byref(t)
    fn = {"trim": lambda p, n: lib.pitch_enqueue_paged_trim(ref, p, n, None),
          "fork": lambda p, n: lib.pitch_enqueue_paged_fork(ref, c, 1, p, n, None),
          "compact": lambda p, n: lib.pitch_enqueue_paged_compact(ref, c, 1, p, n, None, 0, None)}[name]
    size = 4 * (PAGES if name == "compact" else B)
    assert fn(mem(size), size - 4) == BAD and fn(mem(size) + 2, size) == BAD and fn(t.lengths, size) == BAD
    if name != "compact":
        assert fn(None, size) == BAD
    assert "device" not in lib.pitch_last_error().decode()


def test_null_calls(lib):  # noqa: F811
    mem = Memory()
    t, n = _tables(mem), ctypes.c_uint64(0)
    assert lib.pitch_enqueue_prompt_attention(None, None) == BAD
    assert lib.pitch_prompt_attention_workspace_size(None, ctypes.byref(n)) == BAD
    assert lib.pitch_paged_tables_workspace_size(None, ctypes.byref(n)) == BAD
    assert lib.pitch_paged_tables_workspace_size(ctypes.byref(t), None) == BAD
    assert lib.pitch_enqueue_paged_reserve(ctypes.byref(t), None, None) == BAD
    assert lib.pitch_enqueue_paged_reserve(None, None, None) == BAD
    assert lib.pitch_enqueue_paged_fork(ctypes.byref(t), None, 1, mem(64), 64, None) == BAD
