"""The order of calls on the same page tables that are made on different streams, without a GPU: streams and events that keep clocks of
what lies behind them stand for torch's, and every call has to come behind the one before it."""
import threading
import types

import pytest
import torch

import pitch_amd as P
from pitch_amd import paged, pages


class Event:
    def __init__(self, clock):
        self.clock = dict(clock)


class Stream:
    """A stream of torch's (or with `external` a handle that the program made): for each stream the calls that have ended when its
    next one begins."""
    handles = iter(range(16, 1 << 20, 16))

    def __init__(self, external=False):
        self.cuda_stream = next(Stream.handles)
        self.stream_id = self.cuda_stream if external else self.cuda_stream + 3
        self.clock, self.capturing, self.gone = {}, False, False

    def record_event(self):
        assert not self.gone, "an event on a stream that does not exist any more"
        assert not self.capturing, "an event of a capture, which eager work must not wait for"
        return Event(self.clock)

    def wait_event(self, event):
        assert not self.capturing, "a capture cannot wait for work outside of it"
        for key, at in event.clock.items():
            self.clock[key] = max(self.clock.get(key, 0), at)

    def wait_stream(self, other):
        self.wait_event(other.record_event())


class Device:
    """What the classes ask of torch.cuda."""

    def __init__(self):
        self.Stream, self.Event = Stream, Event
        self.main = Stream()
        self.now, self.known = self.main, {self.main.cuda_stream: self.main}

    def made(self, **more):
        s = Stream(**more)
        self.known[s.cuda_stream] = s
        return s

    def current_stream(self, device=None):
        return self.now

    def default_stream(self, device=None):
        return self.main

    def ExternalStream(self, handle, device=None):  # noqa: N802 (torch's name)
        s = self.known[handle]
        if s.stream_id == handle:
            return s
        made = Stream(external=True)      # the same stream by its handle
        made.cuda_stream = made.stream_id = handle
        made.clock = s.clock
        return made

    def is_current_stream_capturing(self):
        return self.now.capturing

    class _Within:
        def __init__(self, device, stream):
            self.device, self.stream = device, stream

        def __enter__(self):
            self.before, self.device.now = self.device.now, self.stream

        def __exit__(self, *error):
            self.device.now = self.before

    def stream(self, stream):
        return Device._Within(self, stream)


@pytest.fixture
def cuda(monkeypatch, built_library):
    device = Device()
    fake = types.SimpleNamespace(cuda=device, **{n: getattr(torch, n) for n in ("full", "zeros", "empty", "int32", "int64", "uint8", "Tensor")})
    for module in (paged, pages):
        monkeypatch.setattr(module, "_torch", lambda: fake)
        monkeypatch.setattr(module, "_flat", lambda t, name, dtype, count: (None, 0) if t is None else (t.data_ptr(), t.nbytes))
        monkeypatch.setattr(module, "_tables", lambda t: (t.data_ptr(), t.nbytes))
    monkeypatch.setattr(paged, "_buf", lambda t, name: (t.data_ptr(), t.nbytes))
    monkeypatch.setattr(paged, "_stream_handle", lambda stream, d=None: device.now.cuda_stream if stream is None else stream
                        if isinstance(stream, int) else stream.cuda_stream)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: None)
    return device


class Program:
    """Tables, and calls on them that are checked for their order in place of being launched."""

    def __init__(self, cuda):
        from pitch_amd import _lib
        cache = object.__new__(P.PagedCache)
        cache.pitch = types.SimpleNamespace(device=torch.device("cpu"), _lib=_lib.load())
        cache.pages, cache.pageSize, cache._cstruct = 8, 16, _lib.PitchPagedCacheC()
        self.cuda, self.count, self.last = cuda, 0, {}
        self.tables = P.PagedTables(cache, sequences=2, width=3)
        self.calls = [P.PagedTrim(self.tables, torch.zeros(2, dtype=torch.int32)), P.PagedFork(self.tables, torch.zeros(2, dtype=torch.int32))]
        for call in self.calls:
            call._launch = self.launch

    def launch(self, handle):
        stream = self.cuda.known[handle]
        if stream.capturing:
            return 0
        for key, at in self.last.items():
            assert stream.clock.get(key, 0) >= at, "a call does not wait for the one before it"
        self.count += 1
        stream.clock[handle] = self.count
        self.last = {handle: self.count}
        return 0

    def capture(self, stream):
        """A capture begins, as torch.cuda.graph does it: behind all work of the device."""
        stream.capturing, self.last = True, {}

    def call(self, stream=None):
        self.calls[self.count % 2].enqueue(stream)


def test_calls_in_turn_on_two_streams(cuda):
    p, side = Program(cuda), cuda.made()
    for _ in range(3):
        p.call()
        p.call(side)
        p.call(side)
    p.call(side.cuda_stream)
    p.call()
    with cuda.stream(side):
        p.call()
    p.call()
    assert p.count == 13


def test_calls_on_many_streams(cuda):
    p, streams = Program(cuda), [cuda.made() for _ in range(4)] + [cuda.made(external=True) for _ in range(2)]
    for i in range(60):
        s = streams[i * i % 7 % 6]
        p.call(s if i % 3 else s.cuda_stream)
    assert p.count == 60


def test_a_stream_of_the_program_may_be_gone_before_the_next_call(cuda):
    """Nothing is asked of such a stream but by a call on it."""
    for form in ("stream", "handle", "current"):
        p, side = Program(cuda), cuda.made(external=True)
        p.call()
        if form == "current":
            with cuda.stream(side):
                p.call()
        else:
            p.call(side if form == "stream" else side.cuda_stream)
        side.gone = True
        p.call()
        p.call(cuda.made())
        assert p.count == 4


def test_a_capture_neither_waits_nor_is_waited_for(cuda):
    p, side, graph = Program(cuda), cuda.made(), cuda.made()
    p.call()
    p.capture(graph)
    with cuda.stream(graph):
        p.call()
    p.call(side)          # (another thread's eager call, or one in a relaxed capture)
    graph.capturing = False
    p.call(graph)
    p.capture(graph)
    p.call(side)
    p.call()
    assert p.count == 5


def test_calls_of_several_threads(cuda):
    """Looking for the last call and making the next one is one step."""
    p, streams = Program(cuda), [cuda.made() for _ in range(4)]
    errors, inside = [], threading.Lock()
    launch = p.launch

    def slow(handle):
        assert inside.acquire(blocking=False), "two calls are made at once"
        try:
            threading.Event().wait(0.001)
            return launch(handle)
        finally:
            inside.release()

    for call in p.calls:
        call._launch = slow

    def work(stream):
        try:
            for _ in range(10):
                p.call(stream)
        except BaseException as e:  # noqa: BLE001 (told to the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    assert p.count == 40
