"""attention_tree_forward where the running maximum moves: lanes of one wave whose maximum
grows a little, much, in late stages alone, in every stage, or is found there first.

Queries are along one of eight directions, whose keys peak along the context by a schedule
of their own: a score in powers of two is what the key holds in that dim.  Partitions are
long: as many sequences and heads as fill the GPU.  The bound of an output is that of
test_gpu_tree_attention.py; a move of the maximum scales sums and outputs by the same
factor and rounds each once, 2^-24, at most once per stage: 44 more to the sum's."""
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import ancestors, random_tree

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")
KVH, GROUP, SEQS, STAGES = 8, 2, 32, 40


def schedule(direction, stage):
    """The peak of a direction's keys in a stage, in powers of two."""
    return [0, 6 * (stage >= 9), 9 * (stage >= 30), 9 * ((stage >= 3) + (stage >= 17) + (stage >= 33)),
            100 * (stage >= 2), 40 - stage, 3 * stage, 9 * (stage >= STAGES - 1)][direction]


@pytest.mark.parametrize("rows", [5, 64])
@pytest.mark.parametrize("out16", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_maxima_that_grow(backend, dim, out16, rows):
    stage = 8192 // dim
    rng = np.random.default_rng(dim + rows)
    contexts = [stage * STAGES - int(rng.integers(0, stage)) for _ in range(SEQS)]
    contexts[3] = 3  # (almost) all keys are the tree's
    trees = [random_tree(rng, rows, 9)[0] for _ in range(SEQS)]
    most = max(contexts) + rows
    pool = pkg.KvCache(backend, KVH, dim, 16, SEQS * (most // 16 + 2), most, SEQS, page_order_seed=3)
    g = torch.Generator().manual_seed(rows)
    cached = []
    for n in contexts:
        k = 0.25 * torch.randn((n, KVH, dim), generator=g)
        v = torch.randn((n, KVH, dim), generator=g)
        for s in range(-(-n // stage)):
            for h in range(KVH):
                for d in range(8):
                    at = s * stage + int(rng.integers(0, stage))
                    if at < n:
                        k[at, h, 2 + d] += schedule(d, s)
        k, v = k.bfloat16(), v.bfloat16()
        pool.append(pool.open(), k.reshape(n, -1).cuda(), v.reshape(n, -1).cuda())
        cached.append((k.cuda().double(), v.cuda().double()))
    total = SEQS * rows
    # (dims 0 and 1 are rotated, and 0)
    q = 0.02 * torch.randn((total, KVH * GROUP, dim), generator=g)
    along = torch.randint(0, 8, (total, KVH * GROUP, 1), generator=g)
    q.scatter_add_(2, along + 2, torch.full(along.shape, math.sqrt(dim) * math.log(2)))
    q[..., :2] = 0
    k, v = (torch.randn((total, KVH, dim), generator=g) for _ in range(2))
    k[..., :2] = 0
    positions = torch.tensor([[n + len(ancestors(t, r)) - 1] * 3 for n, t in zip(contexts, trees)
                              for r in range(rows)], dtype=torch.int32)
    out = torch.full((total, KVH * GROUP * dim), math.nan, device="cuda",
                     dtype=torch.bfloat16 if out16 else torch.float32)
    pkg.attention_tree_forward(backend, pool, list(range(SEQS)), [rows] * SEQS, [p for t in trees for p in t],
                               q.reshape(total, -1).cuda(), k.reshape(total, -1).cuda(), v.reshape(total, -1).cuda(),
                               positions.cuda(), out, heads=KVH * GROUP, kv_heads=KVH, head_dim=dim, rotary_dim=2,
                               rope_theta=1e4)
    worst = 0.0
    for i, (n, tree) in enumerate(zip(contexts, trees)):
        at = slice(i * rows, (i + 1) * rows)
        keys = torch.cat([cached[i][0], k[at].bfloat16().cuda().double()])
        values = torch.cat([cached[i][1], v[at].bfloat16().cuda().double()])
        hidden = torch.zeros((rows, n + rows), dtype=torch.bool)
        hidden[:, n:] = True
        for r in range(rows):
            hidden[r, [n + a for a in ancestors(tree, r)]] = False
        hidden = hidden.cuda()
        # [kv head][row x head of it]
        qs = q[at].cuda().double().view(rows, KVH, GROUP, dim).permute(1, 0, 2, 3).reshape(KVH, rows * GROUP, dim)
        hide = hidden[:, None].expand(rows, GROUP, -1).reshape(1, rows * GROUP, -1)
        ks, vs = (x.permute(1, 2, 0).contiguous() for x in (keys, values))
        score = (torch.bmm(qs, ks) / math.sqrt(dim)).masked_fill(hide, -math.inf)
        p = torch.softmax(score, -1)
        vs = vs.transpose(1, 2).contiguous()
        want, size = torch.bmm(p, vs), torch.bmm(p, vs.abs())
        big = (torch.bmm(qs.abs(), ks.abs()) / math.sqrt(dim)).masked_fill(hide, 0.0).amax(-1, keepdim=True)
        ds = big * ((32 + dim) * 2.0 ** -24 + (2.0 ** -16 if out16 else 2.0 ** -24))
        tol = size * (2 * ds + (2.0 ** -8 if out16 else 2.0 ** -22) + (n + rows + 64 + 44) * 2.0 ** -24)
        if out16:
            tol = tol + 2.0 ** -8 * (want.abs() + tol)
        got = out[at].double().view(rows, KVH, GROUP, dim).permute(1, 0, 2, 3).reshape(KVH, rows * GROUP, dim)
        assert torch.isfinite(got).all()
        worst = max(worst, float(((got - want).abs() / tol).max()))
    assert worst <= 1.0, f"error {worst:.2f} times the bound"
    pool.destroy()


@pytest.mark.parametrize("out16", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_scores(backend, dim, out16):
    """Scores of several hundred, contexts of none to many stages."""
    from test_gpu_tree_attention import Case

    rng = np.random.default_rng(4)
    trees = [random_tree(rng, n)[0] for n in (9, 40, 100)]
    case = Case(backend, 4, 4, 2, dim, dim, trees, [700, 0, 33], norm=False, scale=20.0, out16=out16)
    case.check(case.run())
    case.pool.destroy()
