"""attention_tree_forward with keys and values that are not finite: a row sees its own
ancestors alone, so the other rows keep their bits, and the call reports the error."""
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import Case, ancestors, random_tree

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")

LARGE_NAN = np.uint32(0x7fffffff).view(np.float32)  # (rounded as a number it would be -0)
SHAPES = {64: (6, 2, 64), 128: (8, 2, 128), 256: (4, 2, 256), 80: (4, 2, 80)}


def run(case):
    """The outputs of an asynchronous call as [row][head][dim], and whether it reports an
    error.  The drafts are taken back."""
    out = torch.full((case.rows, case.heads * case.dim), math.nan, device="cuda",
                     dtype=torch.bfloat16 if case.out16 else torch.float32)
    args = [t.cuda() for t in (case.q, case.k, case.v, case.pos)]
    gains = [g.cuda() for g in case.gains] if case.norm else [None, None]
    torch.cuda.synchronize()
    pkg.attention_tree_forward(
        case.backend, case.pool, case.ids, [len(t) for t in case.trees], [p for t in case.trees for p in t], *args,
        out, heads=case.heads, kv_heads=case.kvh, head_dim=case.dim, rotary_dim=case.rot, rope_theta=case.theta,
        q_norm=gains[0], k_norm=gains[1], gated=case.gated, norm_offset=case.gated, asynchronous=True)
    error = False
    try:
        case.backend.synchronize()
    except pkg.PluginError as e:
        assert "non-finite" in str(e) or "not finite" in str(e)
        error = True
    for i, c in zip(case.ids, case.contexts):
        case.pool.truncate(i, c)
    return out.cpu().float().numpy().reshape(case.rows, case.heads, case.dim), error


@pytest.mark.parametrize("context", [0, 40, 3000])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("out16", [False, True])
@pytest.mark.parametrize("dim", list(SHAPES))
def test_bad_rows(backend, dim, out16, norm, context):
    heads, kvh, rot = SHAPES[dim]
    tree = random_tree(np.random.default_rng(dim), 45, 7)[0]
    tree[:6] = [-1, 0, 0, -1, 2, 1]
    tree[17], tree[44] = 5, 3
    case = Case(backend, 3, heads, kvh, dim, rot, [tree, [-1, 0, 0]], [context, 70], norm=norm, bf16=out16, out16=out16)
    clean, error = run(case)
    assert not error and np.all(np.isfinite(clean))
    for row, value, where in ((1, math.inf, "v"), (1, math.nan, "v"), (5, -math.inf, "k"), (1, math.nan, "k"),
                              (44, math.inf, "v"), (44, math.nan, "k"), (0, math.nan, "v"), (5, 3.4e38, "v"), (5, LARGE_NAN, "v")):
        tensor = case.v if where == "v" else case.k
        at = dim + 3  # of the second KV head
        kept = tensor[row, at].clone()
        tensor[row, at] = torch.tensor(value).to(tensor.dtype)
        got, error = run(case)
        tensor[row, at] = kept
        below = [r for r in range(len(tree)) if row in ancestors(tree, r)]
        others = [r for r in range(case.rows) if r not in below]
        assert error
        assert np.array_equal(got[others], clean[others])
        assert np.array_equal(got[below, :heads // 2], clean[below, :heads // 2])
        assert not np.any(np.isfinite(got[below, heads // 2:]))
    assert np.array_equal(run(case)[0], clean)
    case.pool.destroy()


@pytest.mark.parametrize("dim", list(SHAPES))
def test_bad_queries(backend, dim):
    """A query that is not finite is its own row's and head's."""
    heads, kvh, rot = SHAPES[dim]
    tree = random_tree(np.random.default_rng(1), 20, 7)[0]
    case = Case(backend, 3, heads, kvh, dim, rot, [tree], [100], norm=False)
    clean, _ = run(case)
    case.q[2, dim + 1] = math.nan
    got, _ = run(case)
    assert not np.any(np.isfinite(got[2, 1]))
    got[2, 1] = clean[2, 1]
    assert np.array_equal(got, clean)
    case.pool.destroy()
