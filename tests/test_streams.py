"""What the host layer asks about streams (runs without a GPU)."""

from __future__ import annotations

import gc
import weakref

import pytest

from mmfp4 import _lib


def test_the_default_stream_is_in_no_capture():
    assert _lib.load().mm_capture_id(None) == 0


def test_counters_are_cleared_in_a_whole_workspace():
    for ws, size in ((None, 1 << 20), (8, 1 << 20), (16, 65535)):
        with pytest.raises(ValueError, match="16-byte aligned"):
            _lib.call("mm_clear_counters", ws, size, None)


class Stream:
    def __init__(self, raw):
        self.raw, self.waits = raw, []

    def wait_event(self, event):
        self.waits.append(event)


class Event:
    done = False
    cuda_event = 1

    def record(self, stream):
        self.made_on = stream.raw


class Array:
    """As much of a device tensor as the cache of derived copies looks at."""
    is_cuda, dtype, shape = True, "words", (3,)

    def __init__(self):
        self._version, self.recorded = 0, []

    def data_ptr(self):
        return id(self)

    def get_device(self):
        return 0

    def record_stream(self, stream):
        self.recorded.append(stream.raw)


class Machine:
    """The current stream, whether it is being captured, and the events of this process."""

    def __init__(self, monkeypatch):
        self.stream, self.capturing, self.events = Stream(1), False, []

        def event():
            self.events.append(Event())
            return self.events[-1]
        lib = type("Lib", (), {"mm_event_done": lambda _, e: self.events[-1].done})()
        monkeypatch.setattr(_lib, "load", lambda: lib)
        monkeypatch.setattr(_lib, "_raw_stream", lambda index: self.stream.raw)
        monkeypatch.setattr("torch.cuda.Event", event)
        monkeypatch.setattr("torch.cuda.current_stream", lambda index=None: self.stream)
        monkeypatch.setattr("torch.cuda.is_current_stream_capturing", lambda: self.capturing)


@pytest.fixture
def machine(monkeypatch):
    return Machine(monkeypatch)


def derive(src, built):
    def build(s):
        built.append(Array())
        return built[-1]
    return _lib.derived(src, "padded", build)


def test_another_stream_waits_for_a_derived_copy(machine):
    src, built = Array(), []
    first = derive(src, built)
    assert derive(src, built) is first and not machine.stream.waits and not first.recorded
    other = machine.stream = Stream(2)
    assert derive(src, built) is first and len(built) == 1
    assert other.waits == machine.events and first.recorded == [2]
    machine.events[0].done = True
    machine.stream = Stream(3)                    # there by now: nothing to wait for
    assert derive(src, built) is first
    assert not machine.stream.waits and first.recorded == [2, 3]


def test_a_copy_made_under_capture_is_not_kept(machine):
    src, built = Array(), []
    machine.capturing = True
    inside = derive(src, built)
    machine.capturing = False
    outside = derive(src, built)
    assert outside is not inside and derive(src, built) is outside and len(built) == 2


def test_capture_uses_a_copy_that_is_known_to_be_there(machine):
    src, built = Array(), []
    kept = derive(src, built)
    machine.capturing = True
    assert derive(src, built) is not kept         # a replay would not wait for its making
    machine.events[0].done = True
    assert derive(src, built) is kept
    machine.capturing = False
    alive = weakref.ref(kept)
    src._version += 1                             # written in place: a new copy, and the graph's
    assert derive(src, built) is not kept
    built.clear()
    del kept
    assert alive() is not None
    del src
    gc.collect()
    assert alive() is None and not _lib._made
