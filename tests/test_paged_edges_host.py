"""Host side of the rotary, paged-cache and logit operators at their edges (no GPU): a library that only records its calls."""

import ctypes
import math
import threading

import numpy as np
import pytest

from minifield_training_b200 import _lib, device
from minifield_training_b200.device import DeviceArray


class FakeDevice:
    """Answers the runtime calls: memory is a counter, streams have the ids given to them, nothing else runs."""

    def __init__(self):
        self.calls, self.packed, self.next, self.freed = [], [], 1 << 20, []
        self.current, self.ids, self.capturing = 0, {}, set()

    def call(self, name, *args):
        self.calls.append((name, args))
        if name == "mfb_malloc":
            args[0]._obj.value = self.next
            self.next += -(-int(args[1]) // 256) * 256
        elif name == "mfb_stream_identity":
            handle = getattr(args[0], "value", args[0])
            args[1][0], args[1][1] = self.current, self.ids.get((self.current, handle), handle or 1)
            if handle in self.capturing:
                args[1][1] = 0

    def call_packed(self, name, flags, *args, stream=None):
        self.packed.append((name, args))

    def names(self):
        return [name for name, _ in self.calls]


@pytest.fixture
def fake(monkeypatch):
    f = FakeDevice()
    monkeypatch.setattr(_lib, "call", f.call)
    monkeypatch.setattr(_lib, "call_packed", f.call_packed)
    monkeypatch.setattr(DeviceArray, "__del__", lambda self: f.freed.append(self.ptr) if self._owner else None)
    monkeypatch.setattr(device, "_STREAM_WORKSPACES", {})
    return f


def array(shape, dtype, ptr=1 << 20):
    return DeviceArray(shape, dtype, ptr=ptr, owner=False)


def test_stream_workspaces_are_kept_per_device_stream_and_thread(fake):
    def get(stream=None, nbytes=1000):
        return device.stream_workspace("w", nbytes, stream)

    first = get()
    assert get() is first and get(stream=0) is first and get(stream=ctypes.c_void_p(1)) is first  # one stream
    assert get(stream=64) is not first
    fake.current = 1
    other = get()  # the default stream's handle is the same on every device
    assert other is not first and get() is other and get(stream=64) is not other
    fake.current = 0
    assert get() is first
    mine, theirs = get(stream=2), []
    thread = threading.Thread(target=lambda: theirs.append(get(stream=2)))
    thread.start()
    thread.join()
    assert get(stream=2) is mine and theirs[0] is not mine


def test_a_reused_stream_handle_gets_a_new_workspace(fake):
    old = device.stream_workspace("w", 1000, 64)
    fake.ids[0, 64] = 7  # the handle's stream was destroyed (its work may still run), a new one has the handle
    new = device.stream_workspace("w", 1000, 64)
    assert new is not old and device.stream_workspace("w", 1000, 64) is new
    fake.capturing.add(64)
    for nbytes in (10, 5000):
        with pytest.raises(ValueError, match="its own workspace"):
            device.stream_workspace("w", nbytes, 64)
