"""gdn_tree_forward with rows that are not finite, and decays of exactly 0: every row
depends on its own ancestors alone.

The recurrence in 64 bits, row by row along each path, says which values are finite;
those are held to it by the tolerance of test_gpu_gdn_tree.py (1e-4 (1 + |x|)), and to the
bits of a call without the bad values: what a masked row adds is 0.  Behind a bad row a
head of a row has values that are not finite where the recurrence's has: not all the same
ones, as an infinite value makes the norm's variance infinite, which divides the others to
0, or NaN with an infinity of the other sign in its sum, and which sums hold both signs
goes by the form of the sum (a state row by row, or S0 and pairs of rows)."""
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


def bad_heads(case, x):
    return np.any(~np.isfinite(x.reshape(case.rows, case.hv, case.dv)), -1)


# the bad value's tensor, and its channel (of qkv: in q, k or v of the first head)
PLACES = {"q": (0, lambda c: 3), "k": (0, lambda c: c.hk * c.dk + 5), "v": (0, lambda c: 2 * c.hk * c.dk + 7),
          "z": (1, lambda c: 2), "a": (2, lambda c: 1), "b": (3, lambda c: 0)}


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("place", list(PLACES))
@pytest.mark.parametrize("widths", WIDTHS)
def test_one_bad_row(backend, widths, place, value):
    tree = random_tree(np.random.default_rng(5), 41, 9)[0]
    tree[:6] = [-1, 0, 0, -1, 2, 1]
    tree[17], tree[18], tree[40] = 5, 2, 17
    case = Case(backend, 5, *widths, [tree, tree[:6]])
    clean, error = run(case)
    assert not error
    which, channel = PLACES[place]
    case.inputs[which][1, channel(case)] = value
    got, error = run(case)
    want, after = exact(case)
    fine = np.isfinite(want)
    below = [r for r in range(len(tree)) if r == 1 or (tree[r] >= 0 and 1 in path(tree, r))]
    others = [r for r in range(case.rows) if r not in below]
    assert np.all(fine[others]) and len(below) > 1
    assert np.array_equal(got[others], clean[others])
    if value != 3e38:  # (squares past f32: finite in 64 bits alone)
        assert np.array_equal(bad_heads(case, got), bad_heads(case, want))
        if np.all(fine):
            assert close(got, want) and not error
        else:
            assert error or place == "z"
        check_paths(case, after, [0, 2, 3, 1, below[-1], len(tree) - 1])
    case.pool.destroy()


def path(tree, r):
    rows = []
    while r >= 0:
        rows.append(r)
        r = tree[r]
    return rows


@pytest.mark.parametrize("widths", WIDTHS)
@pytest.mark.parametrize("rows", [64, 33, 16, 5])
def test_many_bad_rows(backend, widths, rows):
    """Several bad rows, in every block of rows, siblings of good ones."""
    rng = np.random.default_rng(rows)
    tree = random_tree(rng, rows, 12)[0]
    case = Case(backend, 7, *widths, [tree, [-1, 0, 1]])
    clean, _ = run(case)
    bad = [int(r) for r in rng.choice(rows, 1 + rows // 10, replace=False)]
    for r in bad:
        which, channel = PLACES[str(rng.choice(["k", "v", "a", "b"]))]
        case.inputs[which][r, channel(case)] = math.nan
    got, error = run(case)
    want, after = exact(case)
    fine = np.isfinite(want)
    assert error and not np.all(fine)
    assert not np.any(np.isfinite(got[~fine]))  # (NaN is NaN in any sum)
    assert np.array_equal(got[fine], clean[fine])
    check_paths(case, after, range(0, rows, 3))
    case.pool.destroy()


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
