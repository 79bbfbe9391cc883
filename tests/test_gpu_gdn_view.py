"""GdnState.view on the device: tensors on the pool's memory outlive the pool."""
import gc
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")


def new_pool(backend, seed, sequences=2):
    rng = np.random.default_rng(seed)
    pool = pkg.GdnState(backend, 2, 4, 128, 128, 4, sequences, keep_rows=8)
    held = []
    for i in range(sequences):
        assert pool.open() == i
        held.append((rng.standard_normal((4, 128, 128)).astype(np.float32),
                     rng.standard_normal((pool.channels, 3)).astype(np.float32)))
        pool.write(i, *held[-1])
    return pool, held


def test_view_outlives_the_pool(backend):
    pool, held = new_pool(backend, 1)
    views = [pool.view(i) for i in range(2)]
    row = views[1][0][2, 5]
    pool.destroy()
    del pool
    gc.collect()
    others = [new_pool(backend, seed)[0] for seed in (2, 3)]  # memory that was freed would be theirs
    for (state, history), (m, h) in zip(views, held):
        assert np.array_equal(state.cpu().numpy(), m) and np.array_equal(history.cpu().numpy(), h)
    del views, state, history
    gc.collect()
    assert np.array_equal(row.cpu().numpy(), held[1][0][2, 5])
    for other in others:
        other.destroy()
