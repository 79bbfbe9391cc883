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


@pytest.fixture
def library(monkeypatch):
    lib = Library()

    def as_tensor(array, device=None):
        lib.log.append("tensor")
        return torch.from_numpy(np.asarray(HostArray(array)))

    monkeypatch.setattr(torch, "as_tensor", as_tensor)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: lib.log.append("synchronize"))
    return lib


def new_pool(lib):
    backend = types.SimpleNamespace(lib=lib, context=1, check=lambda status, what: None)
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
