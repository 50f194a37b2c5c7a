"""The paged cache's entry points without a GPU: every argument that can be checked on the host is, before the library looks for
a device. The buffers are host memory and never reach a kernel: a call without a fault of its own stops at the device."""
import ctypes

import pytest

from pitch_amd import _lib

DIM, HEADS, PAGE, PAGES, N, B = 128, 2, 32, 5, 7, 3


@pytest.fixture(scope="module")
def lib(built_library):
    return _lib.load()


class Memory:
    """Host buffers, kept alive, aligned to 64 bytes."""

    def __init__(self):
        self.kept = []

    def __call__(self, nbytes, shift=0):
        raw = (ctypes.c_char * (nbytes + 128))()
        self.kept.append(raw)
        return (ctypes.addressof(raw) + 63) // 64 * 64 + shift


def _config(lib, method=0, dim=DIM, bits=4):
    c = _lib.PitchConfigC()
    c.method, c.dim, c.bits, c.seed = method, dim, bits, 7
    return c


def _cache(lib, mem):
    c = _lib.PitchPagedCacheC()
    c.key_config, c.value_config = _config(lib), _config(lib, bits=3)
    n = PAGES * HEADS * PAGE
    for name, size in (("key_codes", 64), ("key_scales", 4), ("value_codes", 48), ("value_scales", 4)):
        setattr(c, name, mem(n * size))
        setattr(c, name + "_bytes", n * size)
    c.pages, c.page_stride, c.page_size, c.kv_heads, c.layout = PAGES, HEADS * PAGE, PAGE, HEADS, 0
    return c


def _vectors(mem, tokens, heads, esize=2):
    nbytes = tokens * heads * DIM * esize
    return _lib.PitchPagedVectorsC(mem(nbytes), nbytes, heads * DIM, DIM)


def _append(lib, mem):
    c = _lib.PitchPagedAppendC()
    c.io_type, c.q_heads, c.tokens = _lib.IO_BF16, 4, N
    c.keys, c.values = _vectors(mem, N, HEADS), _vectors(mem, N, HEADS)
    c.queries, c.queries_out = _vectors(mem, N, 4), _vectors(mem, N, 4)
    for name, size in (("slots", 8 * N), ("positions", 8 * N), ("query_norm", 2 * DIM), ("key_norm", 2 * DIM)):
        setattr(c, name, mem(size))
        setattr(c, name + "_bytes", size)
    c.cos, c.sin, c.table_bytes, c.rotary_dim, c.eps = mem(4 * 64 * 9), mem(4 * 64 * 9), 4 * 64 * 9, 64, 1e-6
    return c


def _decode(lib, mem):
    c = _lib.PitchPagedDecodeC()
    c.io_type, c.sequences, c.rows, c.table_width = _lib.IO_F16, B, N, 4
    for name, size in (("block_tables", 4 * 4 * B), ("row_starts", 4 * (B + 1)), ("first_tokens", 4 * B)):
        setattr(c, name, mem(size))
        setattr(c, name + "_bytes", size)
    c.keys, c.values = _vectors(mem, N, HEADS), _vectors(mem, N, HEADS)
    return c


def _attention(lib, mem):
    c = _lib.PitchPagedAttentionC()
    c.io_type, c.sequences, c.q_per_kv, c.table_width = _lib.IO_BF16, B, 4, 4
    c.queries, c.output = _vectors(mem, B, 4 * HEADS), _vectors(mem, B, 4 * HEADS)
    for name, size in (("block_tables", 4 * 4 * B), ("lengths", 4 * B), ("slopes", 4 * 4 * HEADS), ("lse", 4 * 4 * HEADS * B)):
        setattr(c, name, mem(size))
        setattr(c, name + "_bytes", size)
    c.scale, c.workspace, c.workspace_bytes = 0.1, mem(1 << 20), 1 << 40
    return c


CALLS = {"append": (_append, "pitch_enqueue_paged_append"), "decode": (_decode, "pitch_enqueue_paged_decode"),
         "attention": (_attention, "pitch_enqueue_paged_attention")}


def _issue(lib, kind, change=lambda cache, call, mem: None):
    mem = Memory()
    make, name = CALLS[kind]
    cache, call = _cache(lib, mem), make(lib, mem)
    change(cache, call, mem)
    rc = getattr(lib, name)(ctypes.byref(cache), ctypes.byref(call), None)
    return rc, lib.pitch_last_error().decode()


@pytest.mark.parametrize("kind", CALLS)
def test_a_whole_call_stops_at_the_device(lib, kind):
    rc, why = _issue(lib, kind)
    assert (rc == _lib.ERR_DEVICE_UNAVAILABLE) or (rc == _lib.ERR_INVALID_INPUT and "not device memory" in why), (rc, why)


def _set(obj, **fields):
    def change(cache, call, mem):
        for path, v in fields.items():
            *way, last = path.split("__")
            at = cache if obj == "cache" else call
            for w in way:
                at = getattr(at, w)
            setattr(at, last, v)
    return change


CACHE_FAULTS = [
    (_set("cache", key_config=_config(None, dim=256), value_config=_config(None, dim=256)), _lib.ERR_INVALID_DIMENSION, "64 or 128"),
    (_set("cache", value_config=_config(None, dim=64)), _lib.ERR_CONFIGURATION_MISMATCH, "differ"),
    (_set("cache", key_config=_config(None, bits=9)), _lib.ERR_INVALID_BIT_WIDTH, "bit width"),
    (_set("cache", key_config=_config(None, method=2)), _lib.ERR_INVALID_INPUT, "method"),
    (_set("cache", page_size=24), _lib.ERR_INVALID_INPUT, "multiple of 16"),
    (_set("cache", page_size=0), _lib.ERR_INVALID_INPUT, "multiple of 16"),
    (_set("cache", page_size=1 << 17), _lib.ERR_INVALID_INPUT, "65536"),
    (_set("cache", kv_heads=0), _lib.ERR_INVALID_INPUT, "KV heads"),
    (_set("cache", layout=2), _lib.ERR_INVALID_INPUT, "layout"),
    (_set("cache", pages=0), _lib.ERR_INVALID_INPUT, "pool"),
    (_set("cache", pages=1 << 28), _lib.ERR_INVALID_INPUT, "pool"),
    (_set("cache", pages=PAGES + 1), _lib.ERR_INVALID_INPUT, "key codes"),
    (_set("cache", page_stride=HEADS * PAGE - 1), _lib.ERR_INVALID_INPUT, "page stride"),
    (_set("cache", page_stride=HEADS * PAGE + 1), _lib.ERR_INVALID_INPUT, "key codes"),
    (_set("cache", page_stride=1 << 63), _lib.ERR_INVALID_INPUT, "page stride"),
    (_set("cache", pages=1 << 26, page_stride=1 << 25), _lib.ERR_INVALID_INPUT, "page stride"),
    (_set("cache", value_scales=None), _lib.ERR_INVALID_INPUT, "value scales"),
    (_set("cache", value_codes_bytes=48 * PAGES * HEADS * PAGE - 1), _lib.ERR_INVALID_INPUT, "value codes"),
]
APPEND_FAULTS = [
    (_set("call", io_type=3), "element type"), (_set("call", tokens=0), "at least 1"),
    (_set("call", tokens=1 << 40), "below 2^31"), (_set("call", tokens=N + 1), "buffer has"),
    (_set("call", keys__data=None), "keys buffer is null"), (_set("call", keys__token_stride=HEADS * DIM + 1), "multiples of 4"),
    (_set("call", values__head_stride=1 << 62), "too large"), (_set("call", values__bytes=N * HEADS * DIM * 2 - 1), "values buffer"),
    (lambda cache, call, mem: setattr(call.keys, "data", call.keys.data + 2), "multiples of 4"),
    (_set("call", queries_out__head_stride=DIM - 2), "overlap"), (_set("call", queries_out__token_stride=0), "overlap"),
    (_set("call", queries_out__data=None), "queries' output"), (_set("call", q_heads=0), "query norm needs queries"),
    (_set("call", slots=None), "slots"), (_set("call", slots_bytes=8 * N - 1), "slots"),
    (lambda cache, call, mem: setattr(call, "slots", call.slots + 4), "aligned"),
    (_set("call", positions_bytes=8), "positions"), (_set("call", positions=None), "need positions"),
    (_set("call", rotary_dim=8), "rotary"), (_set("call", rotary_dim=40), "rotary"), (_set("call", rotary_dim=144), "rotary"),
    (_set("call", table_bytes=4 * 64 - 1), "RoPE cos"), (_set("call", sin=None), "RoPE sin"),
    (_set("call", key_norm_bytes=2 * DIM - 1), "key norm"), (_set("call", query_norm_bytes=0), "query norm"),
    (_set("call", eps=-1.0), "eps"), (_set("call", eps=float("nan")), "eps"), (_set("call", eps=float("inf")), "eps"),
]
DECODE_FAULTS = [
    (_set("call", io_type=7), "element type"), (_set("call", rows=0), "rows"), (_set("call", rows=1 << 31), "rows"),
    (_set("call", sequences=0), "sequences"), (_set("call", sequences=B + 1), "page tables"), (_set("call", table_width=0), "width"),
    (_set("call", table_width=5), "page tables"), (_set("call", row_starts=None), "row starts"),
    (_set("call", row_starts_bytes=4 * B), "row starts"), (_set("call", first_tokens_bytes=4), "first tokens"),
    (_set("call", keys__data=None, values__data=None), "both null"), (_set("call", keys__bytes=64), "keys buffer"),
    (_set("call", keys__head_stride=0), "overlap"), (_set("call", values__token_stride=DIM), "overlap"),
    (_set("call", rows=N + 1), "buffer has"), (_set("call", rows=(1 << 28) + 1), "2^28"),
    (_set("call", keys__token_stride=(1 << 22) + 4, keys__bytes=1 << 40), "token stride"),
    (_set("call", values__token_stride=1 << 23, values__bytes=1 << 40), "token stride"),
]
ATTENTION_FAULTS = [
    (_set("call", io_type=_lib.IO_F32), "float16 or bfloat16"), (_set("call", io_type=9), "element type"),
    (_set("call", sequences=0), "sequences"), (_set("call", sequences=2049), "sequences"), (_set("call", q_per_kv=0), "query heads"), (_set("call", q_per_kv=9), "query heads"),
    (_set("call", q_per_kv=5), "buffer"), (_set("call", sequences=B + 1), "buffer has"),
    (_set("call", output__data=None), "output"), (_set("call", output__token_stride=0), "overlap"),
    (_set("call", queries__head_stride=3), "multiples of 4"), (_set("call", block_tables=None), "page tables"),
    (_set("call", table_width=1 << 40), "width"), (_set("call", lengths_bytes=4 * B - 1), "lengths"),
    (_set("call", slopes_bytes=4), "slopes"), (_set("call", lse_bytes=4), "lse"), (_set("call", scale=float("nan")), "scale"),
    (_set("call", scale=float("inf")), "scale"), (_set("call", softcap=-1.0), "softcap"), (_set("call", softcap=float("nan")), "softcap"),
    (_set("call", window=1 << 31), "window"), (_set("call", table_width=1 << 26, block_tables_bytes=1 << 40), "too many tokens"),
]


@pytest.mark.parametrize("kind", CALLS)
@pytest.mark.parametrize("i", range(len(CACHE_FAULTS)))
def test_cache_faults(lib, kind, i):
    change, code, word = CACHE_FAULTS[i]
    rc, why = _issue(lib, kind, change)
    assert rc == code and word in why, (rc, why)


@pytest.mark.parametrize("kind,i", [(k, i) for k, f in (("append", APPEND_FAULTS), ("decode", DECODE_FAULTS), ("attention", ATTENTION_FAULTS))
                                    for i in range(len(f))])
def test_call_faults(lib, kind, i):
    change, word = {"append": APPEND_FAULTS, "decode": DECODE_FAULTS, "attention": ATTENTION_FAULTS}[kind][i]
    rc, why = _issue(lib, kind, change)
    assert rc == _lib.ERR_INVALID_INPUT and word in why, (rc, why)


def test_null_structs(lib):
    mem = Memory()
    cache = _cache(lib, mem)
    for make, name in CALLS.values():
        fn = getattr(lib, name)
        assert fn(None, ctypes.byref(make(lib, mem)), None) == _lib.ERR_INVALID_INPUT
        assert fn(ctypes.byref(cache), None, None) == _lib.ERR_INVALID_INPUT
    size = lib.pitch_paged_attention_workspace_size
    assert size(None, ctypes.byref(_attention(lib, mem)), None) == _lib.ERR_INVALID_INPUT
    assert size(ctypes.byref(cache), ctypes.byref(_attention(lib, mem)), None) == _lib.ERR_INVALID_INPUT


def test_python_refusals():
    """What the Python classes refuse themselves: tensors that are no device memory."""
    import torch
    import pitch_amd as P
    from pitch_amd import paged
    x = torch.zeros(4, 2, 128)
    with pytest.raises(P.InvalidInput, match="device memory"):
        paged._vectors(x, "keys", 2, 128)
    with pytest.raises(P.InvalidInput, match="torch tensor"):
        paged._vectors([1.0], "keys", 2, 128)
    with pytest.raises(P.InvalidInput, match="device memory"):
        paged._tables(torch.zeros(1, 1, dtype=torch.int32))
    for v in (-1, 1.5, True, "x"):
        with pytest.raises(P.InvalidInput):
            paged._int(v, "window")
