"""gdn_tree_forward at width 128 with sums of few terms: what its products keep of their
operands, below what sums of 128 terms may lose.

The kernel's products of normalised rows with each other and with the state take two fp16
parts of each operand (22 bits); a part that was lost would be 2^-11 of a term.  Conv taps
are (0, 0, 0, 1), so that conv outputs are the inputs; e = 2^-24 below.

An input's silu is off by 2 + |x| log2(e) + 3 of e (the exponent's rounding and its
exponential, a sum, a reciprocal, a product), at most 14 for |x| <= 6; a normalised value
by that, by half of twice it and of the 8 roundings of its squares' sum, and by 4 of the
root and product: 36.  Its parts lose 4 e of it, and 2^-33 where the low part is below the
normal fp16 numbers; a state value's parts 4 e.  A product of three parts is off by the
term that is left out, 4 e, and 3 roundings.
"""
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_gdn_tree import Case
from test_gpu_tree_attention import random_tree

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")
E = 2.0 ** -24
W = 128


def new_case(backend, seed, tree):
    case = Case(backend, seed, 2, 4, W, W, 4, [tree])
    case.inputs[0].clamp_(-6.0, 6.0)
    case.weights[2] = torch.zeros_like(case.weights[2])
    case.weights[2][:, 3] = 1.0
    case.weights[0][:] = -6.0  # (decays near 1: their error is below e)
    return case


def write(case, m):
    case.pool.write(0, m, case.before[0][1])
    case.before[0] = (m, case.before[0][1])


def silu(x):
    return x / (1 + np.exp(-x))


def prepared(case):
    """q, k [row][value head][W], v, the outputs' scale and the steps, in 64 bits."""
    x = silu(case.inputs[0].double().numpy())
    q, k, v = np.split(x, [2 * W, 4 * W], 1)
    q, k = (y.reshape(len(x), 2, W) for y in (q, k))
    q, k = (np.repeat(y / np.sqrt((y * y).sum(-1, keepdims=True) + 1e-6), 2, 1) for y in (q, k))
    scale = case.weights[3].double().numpy() * silu(case.inputs[1].double().numpy()).reshape(-1, 4, W)
    return q, k, v.reshape(-1, 4, W), scale, 1 / (1 + np.exp(-case.inputs[3].double().numpy()))


def check(case, got, size, extra):
    """size: per output the magnitudes behind it before the norm, of which it is off by
    `extra` e at most."""
    want = case.exact()[0].reshape(-1, 4, W)
    scale = prepared(case)[3]
    off = extra * E * size
    unit = np.abs(want / scale)  # o over its root mean square
    rms = size_rms(case)
    # the norm divides by a root that is off by its values' mean, and 16 roundings of its own
    worst = np.sqrt((off ** 2).mean(-1, keepdims=True)) / rms
    tol = np.abs(scale) * (off / rms + unit * (worst + 16 * E)) + np.abs(want) * 16 * E
    err = np.abs(got.reshape(-1, 4, W) - want)
    assert np.all(err <= tol), f"error {(err / tol).max():.2f} times the bound"


def size_rms(case):
    """The root mean square of every row and head's o."""
    out = []
    q, k, v, _, beta = prepared(case)
    states = {-1: case.before[0][0].astype(np.float64)}
    a_log, dt = (x.double().numpy() for x in case.weights[:2])
    a = case.inputs[2].double().numpy()
    for r, p in enumerate(case.trees[0]):
        s = states[p] * np.exp(-np.exp(a_log) * np.logaddexp(0, a[r] + dt))[:, None, None]
        d = beta[r][:, None] * (v[r] - np.einsum("hvk,hk->hv", s, k[r]))
        states[r] = s + np.einsum("hv,hk->hvk", d, k[r])
        o = np.einsum("hvk,hk->hv", states[r], q[r])
        out.append(np.sqrt((o * o).mean(-1, keepdims=True) + W * 1e-6))
    return np.stack(out)


@pytest.mark.parametrize("magnitude", [1e-20, 1.0, 1e10])
def test_state_products(backend, magnitude):
    """One value in every state row, no corrections: an output is one product.  It is off
    by a normalised value's 36 + 4 e, the state's 4, the product's 7, a decay's 2, a root's
    1: 54; and by the low part's 2^-33 = 2^-9 e of the state value."""
    rng = np.random.default_rng(3)
    case = new_case(backend, 3, random_tree(rng, 40, 9)[0])
    case.inputs[3][:] = -math.inf  # (steps of 0)
    m = np.zeros((4, W, W), np.float32)
    at = rng.integers(0, W, (4, W))
    value = (0.5 + rng.random((4, W))) * magnitude
    np.put_along_axis(m, at[..., None], value[..., None].astype(np.float32), 2)
    write(case, m)
    got = case.run()
    q = prepared(case)[0]
    here = np.take_along_axis(q, np.broadcast_to(at, (len(q), 4, W)), 2)
    check(case, got, value * (np.abs(here) + 2.0 ** -9 / 54), 54)
    case.pool.destroy()


@pytest.mark.parametrize("rows", [3, 20, 50])
def test_pair_products(backend, rows):
    """A state of 0, and keys and queries of four values in the same places: a pair's
    product has four terms.  A correction or output adds at most the path's pairs to a
    value; a term is a product of 4 terms, off by 36 + 36 + 8 + 7 + 4 + 2^-7 e of their
    magnitudes, its ratio 4, a step 8, the sums 16 + 4 roundings a row of its path (the
    blocks' inverses among them): 128 e, once more for every correction that it goes
    through: 128 (depth + 1)."""
    rng = np.random.default_rng(rows)
    depth = 4
    tree = random_tree(rng, rows, depth)[0]
    case = new_case(backend, rows, tree)
    few = torch.zeros_like(case.inputs[0][:, :4 * W])
    for head in range(4):  # (2 of q, 2 of k: the same places)
        few[:, head * W + 8 * torch.arange(4) + 3] = 1.0
    case.inputs[0][:, :4 * W] *= few
    write(case, np.zeros((4, W, W), np.float32))
    got = case.run()
    q, k, v, _, beta = prepared(case)
    size, mags = [], {}
    for r, p in enumerate(tree):
        path = []
        while p >= 0:
            path.append(p)
            p = tree[p]
        mags[r] = beta[r][:, None] * (np.abs(v[r]) + sum(
            (np.abs(k[j]) * np.abs(k[r])).sum(-1, keepdims=True) * mags[j] for j in path))
        size.append(sum((np.abs(k[j]) * np.abs(q[r])).sum(-1, keepdims=True) * mags[j] for j in path + [r]))
    check(case, got, np.stack(size), 128 * (depth + 1))
    case.pool.destroy()
