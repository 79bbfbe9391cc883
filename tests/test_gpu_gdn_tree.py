"""gdn_tree_forward and gdn_tree_commit against the recurrence in 64 bits, row by
row along each path.

Tolerance: the outputs are normalised, so a value is about 1; it comes from f32
sums of Dk + Dv + 2 depth terms or fewer (at most 2^9 here for the outputs'
norm, scores and corrections together), each rounding 2^-24 of the sum of
magnitudes, which is within twice the value's scale: 4 * 2^9 * 2^-24 = 1.2e-4;
the framework's f32 tolerance of 1e-4 is used.  A state or history value is
held to 1e-4 of its own scale likewise; history values are inputs, exact.
"""
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import ancestors, random_tree

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")


class Case:
    def __init__(self, backend, seed, hk, hv, dk, dv, conv, trees, *, bf16=False, device=True,
                 decay=16.0, extra_slots=1):
        self.__dict__.update(backend=backend, hk=hk, hv=hv, dk=dk, dv=dv, conv=conv, trees=trees,
                             bf16=bf16, device=device)
        rng = np.random.default_rng(seed)
        self.channels = 2 * hk * dk + hv * dv
        self.pool = pkg.GdnState(backend, hk, hv, dk, dv, conv, len(trees) + extra_slots, keep_rows=64)
        self.ids = [self.pool.open() for _ in trees]
        self.before = []
        for i in self.ids:
            m = 0.2 * rng.standard_normal((hv, dv, dk)).astype(np.float32)
            h = rng.standard_normal((self.channels, conv - 1)).astype(np.float32)
            self.pool.write(i, m, h)
            self.before.append((m, h))
        rows = sum(len(t) for t in trees)
        self.rows = rows
        dtype = torch.bfloat16 if bf16 else torch.float32
        self.inputs = [torch.from_numpy(rng.standard_normal((rows, n)).astype(np.float32)).to(dtype)
                       for n in (self.channels, hv * dv, hv, hv)]
        step = np.exp(math.log(1e-3) + math.log(100) * rng.random(hv))
        self.weights = [torch.from_numpy(x.astype(np.float32)) for x in (
            np.log(1 + (decay - 1) * rng.random(hv)), np.log(np.expm1(step)),
            rng.standard_normal((self.channels, conv)) / 2, 1 + 0.1 * rng.standard_normal(dv))]

    def run(self, asynchronous=False, offset=0):
        def put(t):
            if not self.device:
                return t.numpy()
            # (a tensor that begins `offset` values behind an aligned address)
            whole = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
            whole[offset:].copy_(t.reshape(-1))
            return whole[offset:].view(t.shape)

        out = torch.full((self.rows, self.hv * self.dv), math.nan)
        self.sent = [put(t) for t in self.inputs + self.weights]
        out = put(out)
        pkg.gdn_tree_forward(self.backend, self.pool, self.ids, [len(t) for t in self.trees],
                             [p for t in self.trees for p in t], *self.sent, out,
                             asynchronous=asynchronous)
        if asynchronous:
            self.backend.synchronize()
        return out.cpu().numpy() if self.device else out

    def exact(self, before=None):
        """Outputs, and per sequence and row the state and history after it."""
        qkv, z, a, b = (x.double().numpy() for x in self.inputs)
        a_log, dt, taps, norm = (x.double().numpy() for x in self.weights)
        out, after, at = np.zeros(z.shape), [], 0
        for tree, (m, h) in zip(self.trees, before or self.before):
            states = {-1: (m.astype(np.float64), h.astype(np.float64))}
            for r, p in enumerate(tree):
                s, line = states[p]
                line = np.concatenate([line, qkv[at + r][:, None]], 1)
                x = (line * taps).sum(1)
                x = x / (1 + np.exp(-x))
                q, k, v = np.split(x, [self.hk * self.dk, 2 * self.hk * self.dk])
                q, k = (y.reshape(self.hk, -1) for y in (q, k))
                q, k = (np.repeat(y / np.sqrt((y * y).sum(1, keepdims=True) + 1e-6), self.hv // self.hk, 0)
                        for y in (q, k))
                alpha = np.exp(-np.exp(a_log) * np.logaddexp(0, a[at + r] + dt))
                s = s * alpha[:, None, None]
                miss = v.reshape(self.hv, -1) - np.einsum("hvk,hk->hv", s, k)
                s = s + np.einsum("hv,hk->hvk", miss / (1 + np.exp(-b[at + r]))[:, None], k)
                o = np.einsum("hvk,hk->hv", s, q) / math.sqrt(self.dk)
                o = o / np.sqrt((o * o).mean(1, keepdims=True) + np.float64(np.float32(1e-6))) * norm
                g = z[at + r]
                out[at + r] = o.reshape(-1) * g / (1 + np.exp(-g))
                states[r] = (s, line[:, 1:])
            after.append(states)
            at += len(tree)
        return out, after

    def check_state(self, i, want):
        m, h = self.pool.read(self.ids[i])
        assert np.all(np.abs(m - want[0]) <= 1e-4 * (1 + np.abs(want[0])))
        assert np.array_equal(h, want[1].astype(np.float32))


def close(got, want):
    return np.all(np.abs(got - want) <= 1e-4 * (1 + np.abs(want)))


WIDTHS = [(16, 32, 128, 128, 4), (4, 4, 128, 128, 4), (2, 8, 128, 128, 2), (2, 4, 64, 128, 4),
          (2, 2, 96, 40, 3), (1, 2, 20, 33, 1), (1, 1, 256, 512, 8), (2, 4, 128, 128, 1),
          (3, 6, 128, 128, 5)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("widths", WIDTHS)
def test_tree_and_commit(backend, widths, bf16):
    rng = np.random.default_rng(3)
    trees = [random_tree(rng, n)[0] for n in (1, 19, 6)]
    case = Case(backend, 5, *widths, trees, bf16=bf16)
    got = case.run()
    want, after = case.exact()
    assert close(got, want)
    for i in range(len(trees)):
        case.check_state(i, after[i][-1])  # the forward leaves the states
    rows = [0, 17, 3]
    pkg.gdn_tree_commit(backend, [(case.pool, i, r) for i, r in zip(case.ids, rows)])
    for i, r in enumerate(rows):
        case.check_state(i, after[i][r])
    case.pool.destroy()


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64])
@pytest.mark.parametrize("depth", [1, 5, 64])
def test_rows(backend, rows, depth):
    """Every number of rows; all children of the context, trees, chains."""
    tree = list(range(-1, rows - 1)) if depth == 64 else random_tree(np.random.default_rng(rows), rows, depth)[0]
    case = Case(backend, rows, 2, 4, 128, 128, 4, [tree])
    got = case.run()
    want, after = case.exact()
    assert close(got, want)
    pkg.gdn_tree_commit(backend, [(case.pool, 0, rows - 1)])
    case.check_state(0, after[0][rows - 1])
    case.pool.destroy()


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("widths", [(2, 4, 128, 128, 4), (1, 3, 128, 128, 3), (2, 2, 96, 40, 3)])
def test_tensors_that_begin_anywhere(backend, widths, bf16, offset):
    """Device tensors at any of their values' addresses."""
    rng = np.random.default_rng(offset)
    case = Case(backend, 9, *widths, [random_tree(rng, n)[0] for n in (21, 1, 5)], bf16=bf16)
    got = case.run(offset=offset)
    want, after = case.exact()
    assert close(got, want)
    pkg.gdn_tree_commit(backend, [(case.pool, i, 0) for i in case.ids])
    for i in range(3):
        case.check_state(i, after[i][0])
    case.pool.destroy()


def test_strong_decay(backend):
    """Decays down to e^-100 a row: ratios underflow, never overflow."""
    tree = random_tree(np.random.default_rng(2), 40, 30)[0]
    case = Case(backend, 8, 2, 4, 128, 128, 4, [tree], decay=200.0)
    case.inputs[2] += 1.0
    got = case.run()
    want, _ = case.exact()
    assert np.all(np.isfinite(got)) and close(got, want)
    case.pool.destroy()


@pytest.mark.parametrize("device", [True, False])
def test_many_sequences_and_host_memory(backend, device):
    rng = np.random.default_rng(4)
    trees = [random_tree(rng, int(rng.integers(1, 12)))[0] for _ in range(40)]
    case = Case(backend, 6, 1, 2, 128, 128, 4, trees, device=device)
    got = case.run(asynchronous=device)
    want, after = case.exact()
    assert close(got, want)
    pkg.gdn_tree_commit(backend, [(case.pool, i, len(t) - 1) for i, t in zip(case.ids, trees)],
                        asynchronous=True)
    for i, t in enumerate(trees):
        case.check_state(i, after[i][len(t) - 1])
    case.pool.destroy()


def test_commit_again_and_continue(backend):
    """A sequence is committed to one row, to another, to none, and goes on from the
    committed state: a second tree, then gdn_forward."""
    tree = [-1, 0, 0, 2, -1]
    case = Case(backend, 1, 2, 4, 128, 128, 4, [tree])
    case.run()
    _, after = case.exact()
    for row in (3, 1, -1, 4, 3):
        pkg.gdn_tree_commit(backend, [(case.pool, 0, row)])
        case.check_state(0, after[0][row])
        m, h = case.pool.view(0)
        assert np.array_equal(m.cpu().numpy(), case.pool.read(0)[0])
        assert np.array_equal(h.cpu().numpy(), case.pool.read(0)[1])
    held = case.pool.read(0)
    got = case.run()
    want, after = case.exact([held])
    assert close(got, want)
    pkg.gdn_tree_commit(backend, [(case.pool, 0, 2)])
    case.check_state(0, after[0][2])
    # a chain through gdn_forward gives the same rows
    held = case.pool.read(0)
    case.trees = [[-1, 0, 1, 2, 3]]
    tree_out = case.run()
    out = torch.zeros((5, 4 * 128), device="cuda")
    pkg.gdn_forward(backend, case.pool, case.ids, [5], *case.sent, out)
    assert close(out.cpu().numpy(), tree_out)
    with pytest.raises(pkg.PluginError, match="not a tree call"):
        pkg.gdn_tree_commit(backend, [(case.pool, 0, 2)])
    case.check_state(0, case.exact([held])[1][0][4])
    case.pool.destroy()


def test_commit_over_layers(backend):
    """One commit call for many pools of several widths, more entries than the
    kernel arguments take."""
    cases = [Case(backend, s, 2, 4, dk, dk, 4, [[-1, 0, 1], [-1, -1], [-1, 0]])
             for s, dk in enumerate([128, 128, 64, 30] * 5)]
    wants = []
    for c in cases:
        c.run(asynchronous=True)
        wants.append(c.exact()[1])
    pkg.gdn_tree_commit(backend, [(c.pool, i, r) for c in cases for i, r in zip(c.ids, (2, 1, -1))],
                        asynchronous=True)
    for c, want in zip(cases, wants):
        for i, r in enumerate((2, 1, -1)):
            c.check_state(i, want[i][r])
        c.pool.destroy()


def test_forks_are_apart(backend):
    case = Case(backend, 3, 2, 4, 128, 128, 4, [[-1, 0]])
    case.run()
    fork = case.pool.fork(0)
    pkg.gdn_tree_commit(backend, [(case.pool, 0, 1)])
    assert np.array_equal(case.pool.read(fork)[0], case.before[0][0])
    with pytest.raises(pkg.PluginError, match="not a tree call"):
        pkg.gdn_tree_commit(backend, [(case.pool, fork, 1)])
    case.pool.destroy()


def test_repeats_are_bit_equal(backend):
    tree = random_tree(np.random.default_rng(9), 50)[0]
    case = Case(backend, 2, 4, 8, 128, 128, 4, [tree, tree[:7]])
    outs = [case.run() for _ in range(4)]
    assert all(np.array_equal(outs[0], o) for o in outs[1:])
    case.pool.destroy()


@pytest.mark.parametrize("change,text", [
    (dict(parents=[0, 0]), "parent"),
    (dict(parents=[-1, -3]), "parent"),
    (dict(rows=[0], parents=[]), "empty"),
    (dict(ids=[0, 0], rows=[1, 1], parents=[-1, -1]), "twice"),
    (dict(ids=[5]), "not open"),
    (dict(rows=[65], parents=[-1] * 65), "keep_rows"),
    (dict(eps=0.0), "epsilon"),
])
def test_refusals(backend, change, text):
    case = Case(backend, 1, 2, 4, 128, 128, 4, [[-1, 0]])
    case.run()
    out = torch.zeros((2, 4 * 128), device="cuda")
    with pytest.raises(pkg.PluginError, match=text):
        pkg.gdn_tree_forward(backend, case.pool, change.get("ids", [0]), change.get("rows", [2]),
                             change.get("parents", [-1, 0]), *case.sent, out,
                             eps=change.get("eps", 1e-6))
    pkg.gdn_tree_commit(backend, [(case.pool, 0, 1)])  # the tree before it still counts
    with pytest.raises(pkg.PluginError, match="no such row"):
        pkg.gdn_tree_commit(backend, [(case.pool, 0, 2)])
    with pytest.raises(pkg.PluginError, match="twice"):
        pkg.gdn_tree_commit(backend, [(case.pool, 0, 1), (case.pool, 0, 0)])
    with pytest.raises(pkg.PluginError, match="not open"):
        pkg.gdn_tree_commit(backend, [(case.pool, 1, 0)])
    case.pool.destroy()
