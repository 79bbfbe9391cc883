"""GdnState.view without a GPU: a stub in the library's place, with host memory for the
pool's, whose free is recorded."""
import gc
import importlib
import types

import numpy as np
import pytest
import torch

pkg = importlib.import_module("safetyraise-lmengine_amd")
HV, DV, DK, CHANNELS, TAPS = 2, 3, 4, 2 * 4 + 2 * 3, 3


class Library:
    def __init__(self):
        self.log = []
        self.state = np.arange(HV * DV * DK, dtype=np.float32)
        self.history = np.arange(CHANNELS * TAPS, dtype=np.float32)

    def safetyraise_kernel_gdn_create(self, context, options, handle):
        handle._obj.value = 77
        return 0

    def safetyraise_kernel_gdn_view(self, context, pool, sequence, matrix, history):
        self.log.append("view")
        matrix._obj.value, history._obj.value = self.state.ctypes.data, self.history.ctypes.data
        return 0

    def safetyraise_kernel_gdn_destroy(self, context, pool):
        self.log.append("destroy %d" % pool.value)
        return 0


class HostArray:
    """The same memory for numpy, which keeps this object and so the array's owner."""

    def __init__(self, array):
        self.array = array
        self.__array_interface__ = dict(array.__cuda_array_interface__, version=3)


class Stream:
    def __init__(self, log, handle):
        self.log, self.cuda_stream = log, handle

    def wait_stream(self, other):
        self.log.append("stream %d waits for %d" % (self.cuda_stream, other.cuda_stream))


class Tensor(torch.Tensor):
    """A host tensor that says it is on a GPU."""
    device = None


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    lib.home, lib.current, lib.stream, lib.capturing = 0, 0, 0, False

    def as_tensor(array, device=None):
        x = torch.from_numpy(np.asarray(HostArray(array)))
        there = torch.device(device).index == lib.home
        lib.log.append("tensor" if there else "copy")
        x = (x if there else x.clone()).as_subclass(Tensor)
        x.device = torch.device(device)
        return x

    monkeypatch.setattr(torch, "as_tensor", as_tensor)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: lib.log.append("synchronize"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: lib.capturing)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: lib.current)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 3)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: Stream(lib.log, 0))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(lib.log, lib.stream))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: Stream(lib.log, handle))
    return lib


def new_pool(lib, stream=None):
    backend = types.SimpleNamespace(lib=lib, context=1, stream=stream, check=lambda status, what: None)
    return pkg.GdnState(backend, 1, HV, DK, DV, TAPS + 1, 1, keep_rows=4)


def test_memory_stays_under_a_view(library):
    """The free comes when the last tensor on the memory is gone, once, behind the
    work of the caller's streams."""
    pool = new_pool(library)
    state, history = pool.view(0)
    part = state[1, :, 2:]
    pool.destroy()
    del pool
    gc.collect()
    assert "destroy 77" not in library.log
    del state
    gc.collect()
    assert "destroy 77" not in library.log
    assert part.tolist() == library.state.reshape(HV, DV, DK)[1, :, 2:].tolist()
    del part
    gc.collect()
    assert "destroy 77" not in library.log  # the history is on it too
    assert history[0].tolist() == [0.0, 1.0, 2.0]
    del history
    gc.collect()
    assert library.log[-2:] == ["synchronize", "destroy 77"]
    assert library.log.count("destroy 77") == 1


def test_memory_given_up_under_capture(library):
    """While a graph is captured nothing is waited for or freed: that is left to the next
    pool that is made or destroyed."""
    pool = new_pool(library)
    views = pool.view(0)
    pool.destroy()
    library.capturing = True
    del views
    gc.collect()
    assert "synchronize" not in library.log and "destroy 77" not in library.log
    library.capturing = False
    other = new_pool(library)
    assert library.log[-2:] == ["synchronize", "destroy 77"]
    library.log.clear()
    other.destroy()
    assert library.log == ["destroy 77"]


def test_views_of_a_dropped_pool(library):
    """A pool object that is dropped without destroy leaves its memory."""
    state, history = new_pool(library).view(0)
    gc.collect()
    assert state.shape == (HV, DV, DK) and history.shape == (CHANNELS, TAPS)
    del state, history
    gc.collect()
    assert not [x for x in library.log if x.startswith("destroy")]


def test_destroy_without_views(library):
    pool = new_pool(library)
    pool.destroy()
    assert library.log == ["destroy 77"]
    assert pool.handle is None
    pool.destroy()
    assert library.log == ["destroy 77"]


def test_destroy_after_the_views(library):
    pool = new_pool(library)
    handle = pool.handle
    pool.view(0)
    pool.destroy()
    assert handle.value == 77
    assert library.log[-2:] == ["synchronize", "destroy 77"]


@pytest.mark.parametrize("current,context,want", [
    (0, None, []),  # the default stream and a blocking one
    (5, None, ["stream 5 waits for 0"]),
    (5, 5, []),
    (5, 9, ["stream 5 waits for 9"]),
    (0, 9, ["stream 0 waits for 9"]),
])
def test_callers_stream_waits(library, current, context, want):
    library.stream = current
    new_pool(library, context).view(0)
    assert [x for x in library.log if x.startswith("stream")] == want


@pytest.mark.parametrize("home,current", [(0, 0), (2, 0), (1, 2)])
def test_another_device_is_current(library, home, current):
    """A view is on the pool's memory, not a copy on the current device."""
    library.home, library.current = home, current
    pool = new_pool(library)
    state, history = pool.view(0)
    assert state.device.index == history.device.index == home
    assert state.data_ptr() == library.state.ctypes.data
    assert history.data_ptr() == library.history.ctypes.data


def test_no_view_under_capture(library):
    library.capturing = True
    with pytest.raises(pkg.PluginError, match="cannot be captured"):
        new_pool(library).view(0)
    assert "view" not in library.log
