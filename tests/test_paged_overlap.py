"""Outputs of the paged calls that share memory with what the same call reads or writes: refused on the host, where vectors do
share bytes; slices of one buffer that share none are taken. No GPU: a call without a fault stops at the device."""
import ctypes
import random

import pytest

from pitch_amd import _lib
from test_paged_api import B, DIM, HEADS, N, Memory, _append, _attention, _cache, _decode, lib  # noqa: F401 (a fixture)

Q = 4                    # query heads of an append
ROW = Q + 2 * HEADS      # heads of a fused projection


def _issue(lib, make, name, change):
    mem = Memory()
    cache, call = _cache(lib, mem), make(lib, mem)
    change(call, mem)
    rc = getattr(lib, name)(ctypes.byref(cache), ctypes.byref(call), None)
    return rc, lib.pitch_last_error().decode()


def _stopped_at_the_device(rc, why):
    return rc == _lib.ERR_DEVICE_UNAVAILABLE or (rc == _lib.ERR_INVALID_INPUT and "not device memory" in why)


def _vectors(base, shift, tokens_apart, heads_apart):
    """Vectors of two bytes an element at `shift` elements of a buffer."""
    return _lib.PitchPagedVectorsC(base + 2 * shift, 1 << 30, tokens_apart, heads_apart)


def _append_at(out, queries, keys, values):
    """(shift, token stride, head stride) of each in one buffer, None: in a buffer of its own."""
    def change(call, mem):
        base = mem(1 << 20)
        for name, at in (("queries_out", out), ("queries", queries), ("keys", keys), ("values", values)):
            if at is not None:
                setattr(call, name, _vectors(base, *at))
    return change


FUSED = [(0, ROW * DIM, DIM), (Q * DIM, ROW * DIM, DIM), ((Q + HEADS) * DIM, ROW * DIM, DIM)]           # [token][head]
BY_HEAD = [(0, DIM, N * DIM), (Q * N * DIM, DIM, N * DIM), ((Q + HEADS) * N * DIM, DIM, N * DIM)]                   # [head][token]
TRIPLES = [(i * DIM, 3 * Q * DIM, 3 * DIM) for i in range(3)]                                                       # [token][head][q, k, v]
PARTS = [(i * (DIM + 2), ROW * (DIM + 2), DIM + 2) for i in (0, Q, Q + HEADS)]                                      # padded vectors


@pytest.mark.parametrize("form", [FUSED, BY_HEAD, TRIPLES, PARTS], ids=["fused", "by head", "triples", "padded"])
def test_slices_of_one_buffer_are_taken(lib, form):  # noqa: F811
    q, k, v = form
    assert _stopped_at_the_device(*_issue(lib, _append, "pitch_enqueue_paged_append", _append_at(q, q, k, v)))       # in place
    assert _stopped_at_the_device(*_issue(lib, _append, "pitch_enqueue_paged_append", _append_at(q, None, k, v)))
    wide = (q[0] + 2 ** 16, q[1], q[2])     # behind all of it
    assert _stopped_at_the_device(*_issue(lib, _append, "pitch_enqueue_paged_append", _append_at(wide, q, k, v)))


def _inside(name, shift=0):
    """An input and the queries' output in a buffer of their own."""
    def change(call, mem):
        at = mem(1 << 16) + 4096
        setattr(call, name, at)
        call.queries_out.data = at + shift
    return change


OVERLAPS = [
    (_append_at(FUSED[0], (DIM, ROW * DIM, DIM), None, None), "queries"),                        # one head off
    (_append_at((DIM, ROW * DIM, DIM), None, FUSED[1], FUSED[2]), "keys"),
    (_append_at((3 * DIM, ROW * DIM, DIM), None, None, FUSED[2]), "values"),
    (_append_at((0, Q * DIM, DIM), (DIM * Q, Q * DIM, DIM), None, None), "queries"),              # one token off
    (_append_at((0, Q * DIM, DIM), (0, DIM, N * DIM), None, None), "queries"),                    # in place, transposed
    (_append_at((2, ROW * DIM, DIM), FUSED[0], None, None), "queries"),                           # two elements off
    (_append_at((0, ROW * DIM, DIM), None, (DIM - 2, ROW * DIM, DIM), None), "keys"),
    (_inside("slots"), "slots"), (_inside("query_norm"), "query norm"), (_inside("key_norm", -8), "key norm"),
    (_inside("positions"), "positions"), (_inside("cos", 4), "RoPE cos"), (_inside("sin"), "RoPE sin"),
]


@pytest.mark.parametrize("i", range(len(OVERLAPS)))
def test_append_overlaps(lib, i):  # noqa: F811
    change, word = OVERLAPS[i]
    rc, why = _issue(lib, _append, "pitch_enqueue_paged_append", change)
    assert rc == _lib.ERR_INVALID_INPUT and "overlap" in why and word in why, (rc, why)


def _bytes(base, at, tokens, heads):
    shift, ts, hs = at
    return {2 * (shift + t * ts + h * hs + i) for t in range(tokens) for h in range(heads) for i in range(DIM)}


def test_no_shared_byte_is_taken(lib):  # noqa: F811
    """Random strides: whatever shares a byte is refused; what is taken shares none."""
    rng = random.Random(1)
    refused = taken = 0
    for _ in range(600):
        tokens, heads = rng.randint(1, 3), rng.randint(1, 3)
        out = (2 * rng.randint(0, 300), rng.choice([heads * DIM, heads * DIM + 64, 8 * DIM, 10 * DIM]), rng.choice([DIM, DIM, DIM + 32]))
        keys = (2 * rng.randint(0, 600), rng.choice([out[1], out[1], 2 * DIM, 12 * DIM]), rng.choice([out[2], DIM, 2 * DIM, 3 * DIM]))

        def change(call, mem):
            base = mem(1 << 16)
            call.tokens, call.q_heads = tokens, heads
            call.queries_out, call.keys = _vectors(base, *out), _vectors(base, *keys)
        rc, why = _issue(lib, _append, "pitch_enqueue_paged_append", change)
        if "vectors of the output overlap" in why:
            continue
        shared = _bytes(0, out, tokens, heads) & _bytes(0, keys, tokens, HEADS)
        if _stopped_at_the_device(rc, why):
            taken += 1
            assert not shared, (tokens, heads, out, keys)
        else:
            refused += 1
            assert "queries' output and keys overlap" in why, why
    assert refused > 100 and taken > 100


def _decode_at(keys, values):
    def change(call, mem):
        base = mem(1 << 20)
        call.keys, call.values = _vectors(base, *keys), _vectors(base, *values)
    return change


@pytest.mark.parametrize("keys,values,good", [
    ((0, 2 * HEADS * DIM, DIM), (HEADS * DIM, 2 * HEADS * DIM, DIM), True),                 # [row][keys, values][head]
    ((0, 2 * HEADS * DIM, 2 * DIM), (DIM, 2 * HEADS * DIM, 2 * DIM), True),                 # [row][head][key, value]
    ((0, DIM, N * DIM), (HEADS * N * DIM, DIM, N * DIM), True),
    ((0, HEADS * DIM, DIM), (0, HEADS * DIM, DIM), False),
    ((0, HEADS * DIM, DIM), ((N - 1) * HEADS * DIM, HEADS * DIM, DIM), False),
    ((0, 2 * HEADS * DIM, DIM), (DIM, 2 * HEADS * DIM, DIM), False),
])
def test_read_back_outputs(lib, keys, values, good):  # noqa: F811
    rc, why = _issue(lib, _decode, "pitch_enqueue_paged_decode", _decode_at(keys, values))
    assert _stopped_at_the_device(rc, why) if good else rc == _lib.ERR_INVALID_INPUT and "keys and values overlap" in why, (rc, why)


H = 4 * HEADS   # query heads of an attention


@pytest.mark.parametrize("output,queries,good", [
    ((0, H * DIM, DIM), (0, H * DIM, DIM), True),                   # in place
    ((0, 2 * H * DIM, DIM), (H * DIM, 2 * H * DIM, DIM), True),
    ((0, 2 * H * DIM, 2 * DIM), (DIM, 2 * H * DIM, 2 * DIM), True),
    ((0, H * DIM, DIM), (DIM, H * DIM, DIM), False),                # one head off
    ((0, H * DIM, DIM), (H * DIM, H * DIM, DIM), False),            # one sequence off
    ((0, H * DIM, DIM), (0, DIM, B * DIM), False),                  # the same memory in another order
    ((0, H * DIM, DIM), (0, 0, DIM), False),                        # one sequence's queries for all
])
def test_attention_outputs(lib, output, queries, good):  # noqa: F811
    def change(call, mem):
        base = mem(1 << 20)
        call.output, call.queries = _vectors(base, *output), _vectors(base, *queries)
    rc, why = _issue(lib, _attention, "pitch_enqueue_paged_attention", change)
    assert _stopped_at_the_device(rc, why) if good else rc == _lib.ERR_INVALID_INPUT and "output and query overlap" in why, (rc, why)


def test_attention_lse_in_the_output(lib):  # noqa: F811
    def change(call, mem):
        base = mem(1 << 16)
        call.output, call.lse = _vectors(base, 2048, H * DIM, DIM), base + 4096 + 512
    rc, why = _issue(lib, _attention, "pitch_enqueue_paged_attention", change)
    assert rc == _lib.ERR_INVALID_INPUT and "output and lse overlap" in why, (rc, why)
