"""Calls of the library from several host threads (CPU only, nothing launched)."""

from __future__ import annotations

from _ctypes import FUNCFLAG_PYTHONAPI

from representax_amd import _native as nat


def test_calls_that_enqueue_hold_the_interpreter_lock():
    """A call that gave the lock up would let another thread's launches, over the same
    scratch of the stream, in between its own."""

    lib = nat.load()
    released = {name for name in nat.SIGNATURES
                if not type(getattr(lib, name))._flags_ & FUNCFLAG_PYTHONAPI}
    assert released == {"rpx_check_device_errors"}  # it waits for the device
