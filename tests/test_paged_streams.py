"""A paged cache used on several streams: each call waits for the stream of the last one,
whichever view it came through; nothing waits under capture.

The kernels stand in as in ``test_paged_host``, streams as names.
"""

from __future__ import annotations

import importlib
from contextlib import contextmanager
from unittest.mock import patch

import pytest

torch = pytest.importorskip("torch")

from test_paged_host import _rows, memory  # noqa: E402, F401
import tensorsmith_hip as ts  # noqa: E402
from tensorsmith_hip import nn  # noqa: E402

D = importlib.import_module("tensorsmith_hip.device")


@pytest.fixture
def streams(memory):  # noqa: F811
    """``now``: the current stream; ``order``: what is queued where; ``capturing``: streams that are."""
    class Streams:
        now, capturing, order = 0x10, set(), []

        def __call__(self, name):
            self.now = name
            return self

    state = Streams()
    state.order = order = []

    class Stream:
        def __init__(self, handle, device=None):
            self.handle = handle

        def wait_event(self, event):
            order.append(("wait", self.handle, event.on))

    class Event:
        def record(self):
            self.on = state.now

    @contextmanager
    def on(stream):
        before, state.now = state.now, stream.handle
        try:
            yield
        finally:
            state.now = before

    def noting(name):
        real = getattr(type(memory), name, None)

        def call(*a):
            order.append((name.split("_")[-1], a[-1]))
            return 0 if real is None else real(memory, *a)
        return call

    memory.tsattn_pages4_attend_workspace = lambda *a: 0
    for name in ("append", "apply", "read", "attend"):
        setattr(memory, "tsattn_pages4_" + name, noting("tsattn_pages4_" + name))
    with patch.object(D, "current_stream", lambda dev: state.now), \
            patch.object(torch.cuda, "current_stream", lambda *a: Stream(state.now)), \
            patch.object(torch.cuda, "ExternalStream", Stream), patch.object(torch.cuda, "Event", Event), \
            patch.object(torch.cuda, "stream", on), \
            patch.object(torch.cuda, "is_current_stream_capturing", lambda: state.now in state.capturing):
        yield state


def test_a_page_that_is_taken_again_is_no_longer_read(streams):
    cache = nn.PagedKVCache(2, 2, 32, 100, device="hip", num_pages=2)
    cache.append(_rows([[1.0], [2.0]]), _rows([[1.0], [2.0]]))
    assert {x[1] for x in streams.order} == {0x10}
    streams.order.clear()
    streams(0x20)
    nn.paged_attention(_rows([[1.0]]), cache.rows([0]))
    assert streams.order == [("wait", 0x20, 0x10), ("attend", 0x20)]
    streams.order.clear()
    streams(0x30)
    cache.rows([0]).reset()  # (queues nothing, but what comes after it does)
    cache.rows([1]).append(_rows([[3.0] * 70]), _rows([[3.0] * 70]))
    assert streams.order[0] == ("wait", 0x30, 0x20) and {x[:2] for x in streams.order[1:]} == {
        ("apply", 0x30), ("append", 0x30)}
    streams.order.clear()
    cache.get(), cache.copy(3), cache.compact(3), cache.get()
    assert streams.order and all(x[0] != "wait" and x[1] == 0x30 for x in streams.order)
    streams.order.clear()
    other = cache.copy()
    streams(0x40)
    other.append(_rows([[1.0], [2.0]]), _rows([[1.0], [2.0]]))  # (its pages were written on the other stream)
    assert ("wait", 0x40, 0x30) in streams.order


def test_the_first_call_waits_for_where_the_cache_was_made(streams):
    """The pool's memory may have been freed there a moment ago."""
    cache = nn.PagedKVCache(1, 2, 32, 100, device="hip")
    streams(0x20)
    cache.append(_rows([[1.0]]), _rows([[1.0]]))
    assert streams.order[0] == ("wait", 0x20, 0x10)


def test_nothing_waits_under_capture(streams):
    cache = nn.PagedKVCache(1, 2, 32, 100, device="hip")
    cache.append(_rows([[1.0]]), _rows([[1.0]]))
    streams.order.clear()
    streams(0x20).capturing = {0x20}
    cache.append(_rows([[1.0]]), _rows([[1.0]]))
    assert streams.order == [("append", 0x20)]
    streams(0x10)
    cache.get()
    assert streams.order == [("append", 0x20), ("read", 0x10)]
    streams(0x30).capturing = {0x10}  # (an event recorded there would be the graph's)
    with pytest.raises(RuntimeError, match="is being captured"):
        cache.get()
    streams.capturing = set()
    cache.get()
    assert streams.order[2:] == [("wait", 0x30, 0x10), ("read", 0x30)]


def test_a_captured_call_keeps_its_pages(streams):
    """Cuts that give pages back are refused under capture and change nothing; shorter ones are not."""
    cache = nn.PagedKVCache(3, 2, 32, 100, device="hip", page_size=32)
    cache.append(_rows([[1.0] * 40] * 3), _rows([[1.0] * 40] * 3))
    cache.reorder([0, 0, 2])
    cache.free([2])
    table, refs = cache._core.host.copy(), cache._core.refs.copy()
    streams.capturing = {0x10}
    for call in (cache.reset, lambda: cache.free([0]), lambda: cache.truncate([40, 32, 0]), lambda: cache.rows([1]).reset()):
        with pytest.raises(RuntimeError, match="cannot change while a graph"):
            call()
    assert cache.lengths == (40, 40, 0) and (cache._core.host == table).all() and (cache._core.refs == refs).all()
    cache.truncate([33, 40, 0]), cache.free([2]), cache.free([])
    assert cache.lengths == (33, 40, 0)
    for length in (41, -1):
        with pytest.raises(ValueError, match="truncate length"):
            cache.truncate([33, length, 0])
    streams.capturing = set()
    cache.reset()
    assert cache.pages_in_use == 0


def test_another_devices_capture_is_not_this_ones(memory):  # noqa: F811
    """Page changes go by the stream of the cache's device, whichever device is current."""
    state = {"device": 0, "captured": None}

    @contextmanager
    def on(device):
        before, state["device"] = state["device"], device
        try:
            yield
        finally:
            state["device"] = before

    with patch.object(torch.cuda, "current_device", lambda: state["device"]), patch.object(torch.cuda, "device", on), \
            patch.object(torch.cuda, "is_current_stream_capturing", lambda: state["device"] == state["captured"]):
        cache = nn.PagedKVCache(1, 2, 32, 100, device="hip:1")
        rows = lambda n: ts.Tensor(_rows([[1.0] * n])._data, device="hip:1")  # noqa: E731
        state["captured"] = 0
        cache.append(rows(40), rows(40))
        cache.reset()
        state["captured"] = 1
        for call in (lambda: cache.append(rows(40), rows(40)), cache.compact, cache.copy, lambda: cache.reorder([0])):
            with pytest.raises(RuntimeError, match="cannot change while a graph"):
                call()
