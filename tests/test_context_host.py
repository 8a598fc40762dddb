"""The per-device contexts without a GPU."""
import threading

import pytest

torch = pytest.importorskip("torch")

from webgllm_b200 import q4  # noqa: E402


def test_calls_on_tensors_leave_the_callers_device(monkeypatch):
    """wg_init makes its device the current one; for a call on that device's
    tensors the caller's stays, the first call included."""
    current = [0]

    class Made:
        def __init__(self, device):
            self.device, self.lock, self.handle = device, threading.Lock(), 1
            current[0] = device  # as wg_init does

        enqueue = q4.Context.enqueue

    class Library:
        @staticmethod
        def wg_set_stream(handle, stream):
            return 0

    def set_device(device):
        current[0] = device

    monkeypatch.setattr(q4, "Context", Made)
    monkeypatch.setattr(q4, "_contexts", {})
    monkeypatch.setattr(q4._lib, "lib", lambda: Library)
    monkeypatch.setattr(q4, "_current_device", lambda: current[0])
    monkeypatch.setattr(q4, "_set_device", set_device)
    monkeypatch.setattr(q4, "_raw_stream", lambda device: 0)

    def launch(handle):  # an entry point makes its device current
        current[0] = 1
        return 0

    q4.context_of(1)
    assert current[0] == 0
    q4._contexts.clear()
    q4.context_of(1).enqueue(launch)
    assert current[0] == 0
