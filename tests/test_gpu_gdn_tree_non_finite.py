"""gdn_tree_forward with rows that are not finite, and decays of exactly 0: every row
depends on its own ancestors alone.

The recurrence in 64 bits, row by row along each path, says which values are finite;
those are held to it by the tolerance of test_gpu_gdn_tree.py (1e-4 (1 + |x|)), and to the
bits of a call without the bad values: what a masked row adds is 0.  Behind a bad row no
value is finite where the recurrence's is not."""
import importlib
import math
import warnings

import numpy as np
import pytest
import torch

from test_gpu_gdn_tree import Case, close
from test_gpu_tree_attention import random_tree

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")

WIDTHS = [(2, 4, 128, 128, 4), (1, 2, 128, 128, 7), (2, 4, 64, 40, 4)]


def run(case):
    """The outputs of an asynchronous call, and whether it reports an error."""
    sent = [t.cuda() for t in case.inputs + case.weights]
    out = torch.full((case.rows, case.hv * case.dv), math.nan, device="cuda")
    torch.cuda.synchronize()
    pkg.gdn_tree_forward(case.backend, case.pool, case.ids, [len(t) for t in case.trees],
                         [p for t in case.trees for p in t], *sent, out, asynchronous=True)
    try:
        case.backend.synchronize()
        return out.cpu().numpy(), False
    except pkg.PluginError as e:
        assert "not finite" in str(e)
        return out.cpu().numpy(), True


def exact(case):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return case.exact()


def check_paths(case, after, rows):
    """Commits of rows of sequence 0: finite where the recurrence is."""
    for r in rows:
        pkg.gdn_tree_commit(case.backend, [(case.pool, 0, r)])
        m, h = case.pool.read(0)
        want = after[0][r]
        fine = np.isfinite(want[0])
        assert np.array_equal(np.isfinite(m), fine)
        assert close(m[fine], want[0][fine])
        assert np.array_equal(h, want[1].astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("widths", WIDTHS)
@pytest.mark.parametrize("how", ["a", "a_log"])
def test_decays_of_zero(backend, widths, how):
    """log a of minus infinity: the state before such a row is gone, the rows behind it go
    on from the row."""
    tree = random_tree(np.random.default_rng(6), 30, 9)[0]
    tree[:6] = [-1, 0, 1, 1, 3, 0]
    case = Case(backend, 3, *widths, [tree])
    if how == "a":
        case.inputs[2][1] = math.inf
        case.inputs[2][4] = 3e38
    else:
        case.weights[0][0] = 100.0
    got, error = run(case)
    want, after = exact(case)
    assert np.all(np.isfinite(want)) and not error
    assert np.all(np.isfinite(got)) and close(got, want)
    check_paths(case, after, [1, 2, 4, 0, 5])
    case.pool.destroy()
