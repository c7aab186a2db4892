"""The workspaces that calls keep for a thread, device and stream, over a library that only keeps account (no device)."""
import ctypes
import threading

import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import linear
from seedpack_amd._lib import SpaError

NEED = 1 << 21


class Library:
    """the entry points that the calls under test reach: allocations are numbers, calls are noted"""

    def __init__(self):
        self.device, self.at, self.live, self.need = 0, 1 << 40, {}, NEED
        self.log, self.dead, self.capturing = [], set(), set()

    def __getattr__(self, name):
        if name.endswith("_work_bytes"):
            return lambda *a: self.need
        return lambda *a: self.log.append((name[4:], *a)) or 0

    def spa_get_device(self, d):
        d._obj.value = self.device
        return 0

    def spa_set_device(self, d):
        self.device = d
        return 0

    def spa_malloc(self, p, n):
        self.at += 1 << 30
        self.live[self.at] = (self.device, n)
        p._obj.value = self.at
        return 0

    def spa_free(self, p):
        self.log.append(("free", p))
        del self.live[p]
        return 0

    def spa_stream_synchronize(self, s):
        self.log.append(("stream_synchronize", self.device, s))
        return -3 if s in self.dead else 0

    def spa_stream_is_capturing(self, s, yes):
        yes._obj.value = int(s in self.capturing)
        return 0

    def spa_device_synchronize(self):
        self.log.append(("device_synchronize", self.device))
        return 0

    def work(self):
        """the workspaces of the calls so far"""
        return [c[-3] for c in self.log if c[0] == "project"]

    def freed(self, p):
        return ("free", p) in self.log


@pytest.fixture
def library(monkeypatch):
    L = Library()
    monkeypatch.setattr(dev, "lib", lambda: L)
    monkeypatch.setattr(linear, "lib", lambda: L)
    monkeypatch.setattr(dev, "CACHE", dev._Cache())
    linear.release()
    L.log.clear()
    yield L
    linear.release()
    monkeypatch.undo()


def call(stream=None, **more):
    """one projection on a stream, its result given"""
    at = lambda shape, dtype: dev.DeviceArray(shape, dtype, ptr=4096, owner=dev)
    w = linear.Weight(12, at(8 * 144, np.uint8), 8, 256)
    return linear.project(at((4, 256), np.uint16), w, **{"out": at((4, 8), np.uint16), "stream": stream, **more})


def test_a_workspace_is_kept_for_its_stream(library):
    for s in (None, 7, None, 7, 7):
        call(s)
    a, b = library.work()[:2]
    assert a != b and library.work() == [a, b, a, b, b]
    assert not any(c[0].endswith("synchronize") for c in library.log)


def test_workspaces_are_not_blocks_of_dropped_arrays(library):
    """a dropped array's block may still be in use on another stream"""
    dropped = dev.DeviceArray(NEED, np.uint8)
    at = dropped.ptr
    del dropped
    call(7)
    assert library.work()[0] != at
    library.need = 8 * NEED                                # nor when it grows, and what it grows out of is no array's
    call(7)
    library.need = NEED
    old, new = library.work()
    assert new not in (at, old) and library.freed(old)
    assert dev.DeviceArray(NEED, np.uint8).ptr == at


def test_threads_have_workspaces_of_their_own(library):
    call(7)
    t = threading.Thread(target=call, args=(7,))
    t.start()
    t.join()
    a, b = library.work()
    assert a != b and not library.freed(a)


def test_release_waits_for_devices_and_reaches_every_workspace(library):
    """streams that are gone by now, workspaces of several devices: no handle is called, all memory is back"""
    for d in (0, 1):
        library.device = d
        for s in (None, 7, 8):
            call(s)
    library.dead = {7, 8}
    library.log, calls = [], library.work()
    linear.release()
    assert library.device == 1 and all(library.freed(p) for p in calls)
    assert [c for c in library.log if c[0] == "stream_synchronize"] == []
    first = [c[0] for c in library.log].index("free")
    assert {c[1] for c in library.log[:first] if c[0] == "device_synchronize"} == {0, 1}
    call(8)
    assert library.work()[0] not in calls


def test_a_stream_takes_its_workspaces_with_it(library, monkeypatch):
    """a new stream may get the number of one that has been destroyed: it does not get that one's workspace"""
    monkeypatch.setattr(library, "spa_stream_create", lambda p: setattr(p._obj, "value", 99) or 0, raising=False)
    s = dev.Stream()
    call(s.handle)
    other = threading.Event(), threading.Event()

    def elsewhere():
        call(s.handle)
        other[0].set()
        other[1].wait(10)

    t = threading.Thread(target=elsewhere)
    t.start()
    other[0].wait(10)
    a, b = library.work()
    call(7)
    kept = library.work()[-1]
    del s
    names = [c[0] for c in library.log]
    assert library.freed(a) and library.freed(b) and not library.freed(kept)
    # before the handle can be given again
    assert library.log[-1] == ("stream_destroy", 99) and names.count("free") == 2
    t2 = dev.Stream()
    call(t2.handle)
    assert library.work()[-1] not in (a, b)
    other[1].set()
    t.join()


def test_a_captured_call_brings_its_own_memory(library):
    """a graph keeps the addresses of its capture: neither the kept workspace nor an array made for the result"""
    call(7)
    library.capturing = {7}
    own = dev.DeviceArray(NEED, np.uint8, ptr=1 << 20, owner=dev)
    with pytest.raises(ValueError, match="work"):
        call(7)
    with pytest.raises(ValueError, match="out"):
        call(7, out=None, work=own)
    with pytest.raises(ValueError, match="work"):
        linear.add_squares(dev.DeviceArray((4, 8), np.uint16, ptr=4096, owner=dev), dev.DeviceArray((1, 8), np.float32, ptr=4096, owner=dev),
                           dev.DeviceArray(1, np.int64, ptr=4096, owner=dev), stream=7)
    n = len(library.work())
    call(7, work=own)
    call(8)
    call(None)
    library.need = 0                                       # needs none
    call(7)
    assert len(library.work()) == n + 4 and library.work()[n] == 1 << 20
