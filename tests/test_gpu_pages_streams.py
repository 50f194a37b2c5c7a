"""Calls on the same page tables on streams in turn, without a word from the host between them: each finds what the one before it left."""
import threading

import numpy as np
import pytest
import torch

import pitch_amd as P
from pages_reference import Tables

pytestmark = pytest.mark.gpu
ROWS, WIDTH, PAGE, PAGES = 8, 12, 16, 160


def _i32(a):
    return torch.tensor(np.array(a).copy(), dtype=torch.int32, device="cuda")


def _program(q):
    """Tables over a pool of random bytes, the same in numpy, and a capacity for reserve that every step needs."""
    cache = P.PagedCache(q, q.config("turboQuant", 64, 4), pages=PAGES, pageSize=PAGE, kvHeads=2)
    for t in (cache.keyCodes, cache.valueCodes):
        t.copy_(torch.randint(0, 256, t.shape, device="cuda", dtype=torch.uint8))
    for t in (cache.keyScales, cache.valueScales):
        t.copy_(torch.rand(t.shape, device="cuda"))
    tables = P.PagedTables(cache, sequences=ROWS, width=WIDTH)
    pools = [(t.cpu().numpy(), 2) for t in (cache.keyCodes, cache.keyScales, cache.valueCodes, cache.valueScales)]
    return cache, tables, Tables(np.full((ROWS, WIDTH), -1), np.zeros(ROWS), np.zeros(PAGES), PAGE, pools)


def _steps(rng, tables, ref, n):
    """n calls of each kind in turn, and what their slots and positions have to be (those of the last reserve stand at the end)."""
    calls, want = [], []
    for _ in range(n):
        new, parents = rng.integers(0, 20, ROWS), np.where(rng.random(ROWS) < 0.6, np.arange(ROWS), rng.integers(0, ROWS, ROWS))
        slots, positions = (torch.full((ROWS * 20,), 7, dtype=torch.int64, device="cuda") for _ in range(2))
        calls.append(P.PagedReserve(tables, _i32(new), slots, positions=positions))
        want.append((slots, positions, *ref.reserve(new, ROWS * 20)))
        calls.append(P.PagedFork(tables, _i32(parents)))
        ref.fork(parents)
        keep = ref.lengths - rng.integers(0, 30, ROWS)
        calls.append(P.PagedTrim(tables, _i32(keep)))
        ref.trim(keep)
        calls.append(P.PagedCompact(tables))
        ref.compact()
    return calls, want


def _same(cache, tables, ref, want):
    torch.cuda.synchronize()
    for name, got, right in (("tables", tables.blockTables, ref.tables), ("lengths", tables.lengths, ref.lengths),
                             ("references", tables.references, ref.references)):
        assert np.array_equal(got.cpu().numpy(), right), name
    for got, (right, _) in zip((cache.keyCodes, cache.keyScales, cache.valueCodes, cache.valueScales), ref.pools):
        assert np.array_equal(got.cpu().numpy(), right)
    for slots, positions, s, p in want:
        assert np.array_equal(slots.cpu().numpy(), s) and np.array_equal(positions.cpu().numpy(), p)


@pytest.mark.parametrize("form", ["stream", "handle", "current stream"])
@pytest.mark.parametrize("count", [1, 3])
def test_streams_in_turn(q, form, count):
    """Before each call its stream sleeps for a moment, or does not, so that a call that does not wait would come too early."""
    rng = np.random.default_rng(count)
    cache, tables, ref = _program(q)
    calls, want = _steps(rng, tables, ref, 6)
    streams = [torch.cuda.current_stream()] + [torch.cuda.Stream() for _ in range(count)]
    torch.cuda.synchronize()
    for i, call in enumerate(calls):
        s = streams[i % len(streams)]
        with torch.cuda.stream(s):
            if i % 3 != 1:
                torch.cuda._sleep(2_000_000)
            if form == "current stream":
                call.enqueue()
        if form != "current stream":
            call.enqueue(s if form == "stream" else s.cuda_stream)
    _same(cache, tables, ref, want)


def test_a_stream_of_torchs_costs_its_calls_no_event(q):
    """(An event would cost the host a few microseconds a call.)"""
    _, tables, _ = _program(q)
    s = torch.cuda.Stream()
    for stream in (s, torch.cuda.current_stream()):
        tables.enqueueTrim(_i32(np.zeros(ROWS)), stream=stream)
        assert tables._last_handle == stream.cuda_stream
    torch.cuda.synchronize()


def test_a_graph_between_calls_on_streams(q):
    """A captured step is replayed between eager calls on another stream, which the program orders around it."""
    rng = np.random.default_rng(5)
    cache, tables, ref = _program(q)
    new = _i32(np.zeros(ROWS))
    slots = torch.zeros(ROWS * 20, dtype=torch.int64, device="cuda")
    reserve, side = P.PagedReserve(tables, new, slots), torch.cuda.Stream()
    reserve.enqueue(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reserve.enqueue()
    for _ in range(5):
        n = rng.integers(0, 20, ROWS)
        new.copy_(_i32(n))
        graph.replay()
        right, _ = ref.reserve(n, ROWS * 20)
        keep = ref.lengths - rng.integers(0, 30, ROWS)
        ref.trim(keep)
        k = _i32(keep)
        side.wait_stream(torch.cuda.current_stream())
        tables.enqueueTrim(k, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert np.array_equal(slots.cpu().numpy(), right)
    _same(cache, tables, ref, [])


def test_threads_that_take_turns(q):
    """Calls of two threads, each on a stream of its own, in an order that the host alone gives."""
    rng = np.random.default_rng(6)
    cache, tables, ref = _program(q)
    calls, want = _steps(rng, tables, ref, 4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    turns, errors = [threading.Semaphore(1), threading.Semaphore(0)], []

    def work(me):
        try:
            torch.cuda.set_device(q.device)
            for call in calls[me::2]:
                assert turns[me].acquire(timeout=30)
                with torch.cuda.stream(streams[me]):
                    torch.cuda._sleep(1_000_000)
                call.enqueue(streams[me])
                turns[1 - me].release()
        except BaseException as e:  # noqa: BLE001 (told to the main thread)
            errors.append(e)
            turns[1 - me].release()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    _same(cache, tables, ref, want)
