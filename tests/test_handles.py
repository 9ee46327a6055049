"""The cache of handles (_lib.handle) without a GPU: which handle a call gets, and what keeps one open."""
import gc
import weakref
from collections import OrderedDict

import pytest
import torch


@pytest.fixture
def lib(ge, monkeypatch):
    """_lib with handles that open nothing; lib.stream and lib.capturing are the current stream's."""
    m = ge._lib

    class Handle:
        def __init__(self, device, rows, vocab):
            self.device, self.rows, self.vocab = device, rows, vocab

    monkeypatch.setattr(m, "Handle", Handle)
    monkeypatch.setattr(m, "_handles", OrderedDict())
    monkeypatch.setattr(m, "_captured", set(), raising=False)
    monkeypatch.setattr(m, "_device_handles", {}, raising=False)
    monkeypatch.setattr(m, "stream", 0, raising=False)
    monkeypatch.setattr(m, "capturing", False, raising=False)
    monkeypatch.setattr(m, "raw_stream", lambda device: m.stream)
    monkeypatch.setattr(m, "_capturing", lambda device: m.capturing, raising=False)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    return m


def _gone(ref):
    gc.collect()
    return ref() is None


def test_a_replaced_or_evicted_handle_is_let_go(lib):
    a = weakref.ref(lib.handle(0, 1, 100))
    assert lib.handle(0, 64, 100) is a() and lib.handle(0, 1, 7) is a()
    b = weakref.ref(lib.handle(0, 65, 50))
    assert _gone(a) and (b().rows, b().vocab) == (65, 100)
    for lib.stream in range(1, lib.MAX_HANDLES + 1):
        lib.handle(0, 1, 1)
    assert _gone(b) and len(lib._handles) == lib.MAX_HANDLES


def test_the_handle_of_a_captured_call_stays_open(lib):
    a = weakref.ref(lib.handle(0, 1, 100))
    lib.capturing = True
    assert lib.handle(0, 1, 100) is a()
    lib.capturing = False
    b = weakref.ref(lib.handle(0, 1, 200))  # replaced
    lib.capturing = True
    assert lib.handle(0, 64, 200) is b()
    lib.capturing = False
    for lib.stream in range(1, lib.MAX_HANDLES + 1):  # pushed out
        lib.handle(0, 1, 1)
    assert not _gone(a) and not _gone(b) and (0, 0) not in lib._handles
    lib.release_captured()
    assert _gone(a) and _gone(b)


def test_a_capture_opens_no_handle(lib):
    lib.capturing = True
    with pytest.raises(RuntimeError, match="not open"):
        lib.handle(0, 1, 100)
    lib.capturing = False
    h = lib.handle(0, 1, 100)
    lib.capturing = True
    for rows, vocab in ((65, 100), (1, 101)):
        with pytest.raises(RuntimeError, match="holds 64 of 100"):
            lib.handle(0, rows, vocab)
    assert lib.handle(0, 64, 100) is h and list(lib._handles.values()) == [h]


def test_calls_without_a_workspace_leave_the_streams_handles(lib):
    """Page steps and path moves on any number of streams push no handle out and open none in the streams' cache."""
    a = lib.handle(0, 1, 100)
    d = lib.device_handle(0)
    for lib.stream in range(1, 3 * lib.MAX_HANDLES):
        assert lib.device_handle(0) is d
    assert list(lib._handles.values()) == [a] and d is not a and (d.rows, d.vocab) == (1, 1)
    assert lib.device_handle(1) is not d


def test_a_capture_opens_no_device_handle(lib):
    lib.capturing = True
    with pytest.raises(RuntimeError, match="before the capture"):
        lib.device_handle(0)
    lib.capturing = False
    a = lib.handle(0, 1, 100)
    lib.capturing = True
    assert lib.device_handle(0) is a and not lib._device_handles  # (the stream's, for its error text alone)
    with pytest.raises(RuntimeError):
        lib.device_handle(1)
    lib.capturing = False
    assert lib.device_handle(0) is not a
