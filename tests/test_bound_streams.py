"""A stream that a step has bound is its thread's: operators that another thread calls meanwhile run on that thread's current stream.  No GPU: torch's lookups are stood in for."""
from __future__ import annotations

import threading
from types import SimpleNamespace

from hyperion_b200.ops import native


def test_a_bound_stream_is_its_threads(monkeypatch):
    current = threading.local()
    monkeypatch.setattr(native.torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=current.stream))
    monkeypatch.setattr(native.torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(native.torch._C, "_cuda_getCurrentRawStream", lambda device: current.stream, raising=False)
    bound, looked, found = threading.Event(), threading.Event(), []

    def look():
        return native.stream_ptr().value, native.stream_address()

    def other():
        current.stream = 222
        bound.wait(10)
        found.append(look())
        with native.stream_bound():
            current.stream = 333
            found.append(look())
        found.append(look())
        looked.set()

    thread = threading.Thread(target=other)
    thread.start()
    current.stream = 111
    assert look() == (111, 111)
    with native.stream_bound():
        current.stream = 112
        bound.set()
        assert looked.wait(10)
        assert look() == (111, 111)
        with native.stream_bound():
            assert look() == (112, 112)
        assert look() == (111, 111)
    thread.join()
    assert look() == (112, 112)
    assert found == [(222, 222), (222, 222), (333, 333)]
