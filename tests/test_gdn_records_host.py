"""Which records gdn_tree_commit and gdn_rollback may build from when a launch fails (the
library's host code, without a GPU; its GDN launches compute nothing)."""
import importlib

import numpy as np
import pytest

from host_library import host, host_path  # noqa: F401

pkg = importlib.import_module("safetyraise-lmengine_amd")
SEQS = 40  # more than one launch of a tree call takes


class Layer:
    def __init__(self, backend):
        self.backend = backend
        self.pool = pkg.GdnState(backend, 1, 2, 32, 32, 4, SEQS, keep_rows=4)
        self.ids = [self.pool.open() for _ in range(SEQS)]
        self.weights = [np.zeros(n, np.float32) for n in (2, 2, self.pool.channels * 4, 32)]

    def rows(self, n):
        return [np.zeros((SEQS * n, w), np.float32) for w in (self.pool.channels, 64, 2, 2, 64)]

    def tree(self, parents):
        *x, out = self.rows(len(parents))
        pkg.gdn_tree_forward(self.backend, self.pool, self.ids, [len(parents)] * SEQS, parents * SEQS, *x,
                             *self.weights, out)

    def keep_rows(self, n):
        *x, out = self.rows(n)
        pkg.gdn_forward(self.backend, self.pool, self.ids, [n] * SEQS, *x, *self.weights, out, keep_rows=True)

    def commit(self, seq, row):
        pkg.gdn_tree_commit(self.backend, [(self.pool, seq, row)])


@pytest.mark.parametrize("after", [0, 1])
def test_a_tree_call_fails(host, after):  # noqa: F811
    """Its launches write over the records of the call before: none may be built from."""
    layer = Layer(host)
    layer.tree([-1, 0, 1])
    layer.commit(0, 2)
    host.test.test_fail(b"gdn_tree", after)
    with pytest.raises(pkg.PluginError, match="gdn_tree"):
        layer.tree([-1, -1])
    for seq in (0, SEQS - 1):
        with pytest.raises(pkg.PluginError, match="not a tree call"):
            layer.commit(seq, 1)
    layer.tree([-1, -1])
    layer.commit(0, 1)
    layer.keep_rows(3)
    layer.pool.rollback(5, 1)
    host.test.test_fail(b"gdn_tree", after)
    with pytest.raises(pkg.PluginError, match="gdn_tree"):
        layer.tree([-1, 0])
    with pytest.raises(pkg.PluginError, match="not a KEEP_ROWS call"):
        layer.pool.rollback(5, 2)
    layer.pool.destroy()


def test_a_forward_fails(host):  # noqa: F811
    layer = Layer(host)
    layer.tree([-1, 0, 1])
    host.test.test_fail(b"gdn", 0)
    with pytest.raises(pkg.PluginError, match="gdn"):
        layer.keep_rows(2)
    with pytest.raises(pkg.PluginError, match="not a tree call"):
        layer.commit(3, 1)
    with pytest.raises(pkg.PluginError, match="not a KEEP_ROWS call"):
        layer.pool.rollback(3, 1)
    layer.pool.destroy()
