"""Rounds of speculative decoding with trees of drafts, as a hybrid model runs them:
every layer's tree call, then one kv_compact over the attention layers and one
gdn_tree_commit over the others, on the context's stream without a wait between.

The same tokens are run again as chains (a tree whose rows are the accepted path) on
layers of their own.  Keys and values of a row depend on its inputs and position alone
and come from the same kernel: equal bits.  An output is compared with 1e-3 (1 + |x|):
a score |q k| / 8 is at most about 6 here and carries 32 + 64 roundings of 2^-24, 3.5e-5;
a weight is off by twice that, a value is at most about 4, two computations: 5.6e-4.  A
GDN output or state has the 1e-4 of its own test, twice.
"""
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_tree_attention import ancestors, random_tree

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")
HEADS, KVH, DIM, PAGE = 6, 2, 64, 16
HK, HV, DK, DV, CONV = 2, 4, 128, 128, 4
CHANNELS = 2 * HK * DK + HV * DV


class Layers:
    """Attention and GDN layers of one model, for `seqs` sequences."""

    def __init__(self, backend, seqs, contexts, attention=3, gdn=2, seed=1):
        rng = np.random.default_rng(seed)
        self.backend = backend
        self.kv = [pkg.KvCache(backend, KVH, DIM, PAGE, 160, 1024, seqs + 3, page_order_seed=i + 1)
                   for i in range(attention)]
        self.gdn = [pkg.GdnState(backend, HK, HV, DK, DV, CONV, seqs, keep_rows=64) for _ in range(gdn)]
        for pool in self.kv:
            for c in contexts:
                k, v = (rng.standard_normal((c, KVH * DIM)).astype(np.float32) for _ in range(2))
                s = pool.open()
                if c:
                    pool.append(s, k, v)
        self.weights = []
        for pool in self.gdn:
            for _ in contexts:
                pool.write(pool.open(), 0.2 * rng.standard_normal((HV, DV, DK)).astype(np.float32),
                           rng.standard_normal((CHANNELS, CONV - 1)).astype(np.float32))
            self.weights.append([torch.from_numpy(x.astype(np.float32)).cuda() for x in (
                np.log(1 + 8 * rng.random(HV)), rng.standard_normal(HV) - 3,
                rng.standard_normal((CHANNELS, CONV)) / 2, 1 + 0.1 * rng.standard_normal(DV))])
        self.lengths = list(contexts)

    def verify(self, trees, inputs):
        """Every layer's rows of the trees; inputs: per layer, rows of all sequences."""
        ids, rows = list(range(len(trees))), [len(t) for t in trees]
        parents = [p for t in trees for p in t]
        pos = torch.tensor([[n + len(ancestors(t, r)) - 1] * 3 for n, t in zip(self.lengths, trees)
                            for r in range(len(t))], dtype=torch.int32).cuda()
        outs = [torch.full((sum(rows), n), math.nan, device="cuda")
                for n in [HEADS * DIM] * len(self.kv) + [HV * DV] * len(self.gdn)]
        torch.cuda.synchronize()  # (the tensors are made on another stream)
        for pool, (q, k, v), out in zip(self.kv, inputs[0], outs):
            pkg.attention_tree_forward(self.backend, pool, ids, rows, parents, q, k, v, pos, out,
                                       heads=HEADS, kv_heads=KVH, head_dim=DIM, rotary_dim=DIM,
                                       rope_theta=1e6, asynchronous=True)
        for pool, w, x, out in zip(self.gdn, self.weights, inputs[1], outs[len(self.kv):]):
            pkg.gdn_tree_forward(self.backend, pool, ids, rows, parents, *x, *w, out, asynchronous=True)
        return outs, pos

    def commit(self, trees, accepted):
        """accepted: per sequence a row, or -1."""
        paths = [ancestors(t, r) for t, r in zip(trees, accepted)]
        pkg.kv_compact(self.backend, [(pool, i, i, n, path) for pool in self.kv
                                      for i, (n, path) in enumerate(zip(self.lengths, paths))],
                       asynchronous=True)
        pkg.gdn_tree_commit(self.backend, [(pool, i, r) for pool in self.gdn for i, r in enumerate(accepted)],
                            asynchronous=True)
        self.lengths = [n + len(path) for n, path in zip(self.lengths, paths)]

    def cached(self):
        """All tokens of all layers, by one gather per pool."""
        found = [torch.zeros((sum(self.lengths), KVH * DIM), device="cuda", dtype=torch.bfloat16)
                 for _ in range(2 * len(self.kv))]
        torch.cuda.synchronize()
        for pool, k, v in zip(self.kv, found[::2], found[1::2]):
            pkg.kv_gather(self.backend, [(pool, i, 0, n) for i, n in enumerate(self.lengths)], k, v,
                          asynchronous=True)
        return found

    def destroy(self):
        for pool in self.kv + self.gdn:
            pool.destroy()


def inputs_of(g, rows):
    def randn(n):
        return torch.randn(rows, n, device="cuda", generator=g)

    return ([(randn(HEADS * DIM), randn(KVH * DIM), randn(KVH * DIM)) for _ in range(3)],
            [(randn(CHANNELS), randn(HV * DV), randn(HV), randn(HV)) for _ in range(2)])


def take(inputs, rows):
    return tuple([tuple(t[rows].contiguous() for t in layer) for layer in kind] for kind in inputs)


def test_rounds(backend):
    rng = np.random.default_rng(8)
    contexts = [5, 47, 200, 0]
    model, again = Layers(backend, 4, contexts), Layers(backend, 4, contexts)
    g = torch.Generator(device="cuda").manual_seed(3)
    for turn in range(4):
        trees = [random_tree(rng, int(rng.integers(1, 40)))[0] for _ in contexts]
        accepted = [int(rng.integers(0, len(t))) for t in trees]
        if turn == 1:
            accepted[2] = -1  # nothing of one sequence
        inputs = inputs_of(g, sum(len(t) for t in trees))
        outs, pos = model.verify(trees, inputs)
        model.commit(trees, accepted)
        # the paths as chains (a sequence of which nothing stays runs one row, not kept)
        paths = [ancestors(t, r) if r >= 0 else [0] for t, r in zip(trees, accepted)]
        first = np.cumsum([0] + [len(t) for t in trees])
        rows = torch.tensor([int(first[i]) + r for i, p in enumerate(paths) for r in p])
        chosen = take(inputs, rows.cuda())
        chains = [list(range(-1, len(p) - 1)) for p in paths]
        want, want_pos = again.verify(chains, chosen)
        again.commit(chains, [len(p) - 1 if r >= 0 else -1 for p, r in zip(paths, accepted)])
        found, expected = model.cached(), again.cached()
        backend.synchronize()
        assert model.lengths == again.lengths
        assert torch.equal(pos[rows.cuda()], want_pos)
        for layer, (a, b) in enumerate(zip(outs, want)):
            a = a[rows.cuda()]
            limit = 1e-3 if layer < 3 else 2e-4
            assert torch.all((a - b).abs() <= limit * (1 + b.abs())), (turn, layer)
            assert torch.isfinite(outs[layer]).all()
        for a, b in zip(found, expected):
            assert torch.equal(a, b)
        for a, b in zip(model.gdn, again.gdn):
            for i in range(len(contexts)):
                (m, h), (m2, h2) = a.read(i), b.read(i)
                assert np.all(np.abs(m - m2) <= 2e-4 * (1 + np.abs(m2))) and np.array_equal(h, h2)
    model.destroy()
    again.destroy()


def test_a_fork_keeps_other_tokens(backend):
    """Two targets of one verified sequence keep different paths; both go on."""
    rng = np.random.default_rng(2)
    model = Layers(backend, 1, [70], gdn=0)
    pool = model.kv[0]
    k, v = (rng.standard_normal((9, KVH * DIM)).astype(np.float32) for _ in range(2))
    pool.append(0, k, v)
    a, b = pool.open(), pool.open()
    pkg.kv_compact(backend, [(pool, 0, a, 70, [0, 3, 8]), (pool, 0, b, 70, [1, 2])], asynchronous=True)
    whole, kept_a, kept_b = (pool.read(s)[0] for s in (0, a, b))
    assert np.array_equal(kept_a, whole[list(range(70)) + [70, 73, 78]])
    assert np.array_equal(kept_b, whole[list(range(70)) + [71, 72]])
    pool.append(a, k[:5], v[:5])
    assert np.array_equal(pool.read(0)[0], whole) and np.array_equal(pool.read(b)[0], kept_b)
    model.destroy()


def test_capture_is_refused(backend):
    """Every call refuses while the context's stream captures, and changes nothing."""
    model = Layers(backend, 1, [20], attention=1, gdn=1)
    kv, gdn = model.kv[0], model.gdn[0]
    g = torch.Generator(device="cuda").manual_seed(1)
    inputs = inputs_of(g, 3)
    torch.cuda.synchronize()
    model.verify([[-1, 0, 0]], inputs)
    backend.synchronize()
    state = gdn.read(0)
    k, v = (torch.zeros((2, KVH * DIM), device="cuda") for _ in range(2))
    x = torch.zeros(4, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    q, nk, nv = inputs[0][0]
    pos = torch.zeros((3, 3), dtype=torch.int32, device="cuda")
    out, gout = torch.zeros((3, HEADS * DIM), device="cuda"), torch.zeros((3, HV * DV), device="cuda")
    calls = [
        lambda: pkg.attention_tree_forward(backend, kv, [0], [3], [-1, 0, 0], q, nk, nv, pos, out, heads=HEADS,
                                           kv_heads=KVH, head_dim=DIM, rotary_dim=DIM, rope_theta=1e6,
                                           asynchronous=True),
        lambda: pkg.gdn_tree_forward(backend, gdn, [0], [3], [-1, 0, 0], *inputs[1][0], *model.weights[0], gout,
                                     asynchronous=True),
        lambda: pkg.gdn_tree_commit(backend, [(gdn, 0, 1)], asynchronous=True),
        lambda: pkg.kv_compact(backend, [(kv, 0, 0, 20, [1])], asynchronous=True),
        lambda: pkg.kv_gather(backend, [(kv, 0, 0, 2)], k, v, asynchronous=True),
        lambda: gdn.view(0),
    ]
    texts = []
    torch.cuda.synchronize()
    backend.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            x.add_(1.0)
            for call in calls:
                try:
                    call()
                    texts.append("ran")
                except pkg.PluginError as e:
                    texts.append(str(e))
    finally:
        backend.set_stream(None)
    assert all("cannot be captured" in t for t in texts), texts
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, torch.ones(4, device="cuda"))
    assert kv.len(0) == 23 and np.array_equal(gdn.read(0)[0], state[0])
    for call in calls:  # outside capture the same calls run
        call()
        backend.synchronize()
    assert kv.len(0) == 21
    model.destroy()


@pytest.mark.parametrize("dim,kvh", [(64, 16), (128, 8), (256, 4), (80, 13)])
def test_cache_past_32_bits(backend, dim, kvh):
    """A pool whose last heads begin past 2^31 values and 2^32 bytes gives the results of
    a small one, bit for bit."""
    pages = 2 ** 31 // ((kvh - 1) * 64 * dim) + 64
    rng = np.random.default_rng(dim)
    k, v = (rng.standard_normal((300, kvh * dim)).astype(np.float32) for _ in range(2))
    tree = random_tree(rng, 20)[0]
    g = torch.Generator(device="cuda").manual_seed(dim)
    q, nk, nv = (torch.randn(20, n * dim, device="cuda", generator=g) for n in (2 * kvh, kvh, kvh))
    pos = torch.tensor([[300 + len(ancestors(tree, r)) - 1] * 3 for r in range(20)], dtype=torch.int32).cuda()
    results = []
    for n in (64, pages):
        pool = pkg.KvCache(backend, kvh, dim, 64, n, 1024, 3, page_order_seed=n)
        a, b = pool.open(), pool.open()
        pool.append(a, k, v)
        out = torch.zeros((20, 2 * kvh * dim), device="cuda")
        torch.cuda.synchronize()
        pkg.attention_tree_forward(backend, pool, [a], [20], tree, q, nk, nv, pos, out, heads=2 * kvh,
                                   kv_heads=kvh, head_dim=dim, rotary_dim=dim, rope_theta=1e6)
        pkg.kv_compact(backend, [(pool, a, b, 7, list(range(0, 313, 3)))])
        pkg.kv_compact(backend, [(pool, a, a, 300, ancestors(tree, 19))])
        rows = [np.zeros((pool.len(a) + pool.len(b), kvh * dim), np.float32) for _ in range(2)]
        pkg.kv_gather(backend, [(pool, a, 0, pool.len(a)), (pool, b, 0, pool.len(b))], *rows)
        results.append([out.cpu().numpy(), *rows])
        pool.destroy()
    for small, large in zip(*results):
        assert np.array_equal(small, large)
    assert np.array_equal(results[1][1][:300], torch.from_numpy(k).bfloat16().float().numpy())


def test_states_past_32_bits(backend):
    """The last sequences of a large pool of states and records."""
    seqs = 1500
    pool = pkg.GdnState(backend, 16, 32, 128, 128, 4, seqs, keep_rows=64)
    ids = [pool.open() for _ in range(seqs)]
    rng = np.random.default_rng(5)
    m = 0.2 * rng.standard_normal((32, 128, 128)).astype(np.float32)
    h = rng.standard_normal((8192, 3)).astype(np.float32)
    g = torch.Generator(device="cuda").manual_seed(2)
    tree = random_tree(rng, 25)[0]
    x = [torch.randn(25, n, device="cuda", generator=g) for n in (8192, 4096, 32, 32)]
    w = [torch.rand(32, device="cuda", generator=g), torch.randn(32, device="cuda", generator=g) - 3,
         torch.randn((8192, 4), device="cuda", generator=g) / 2, torch.ones(128, device="cuda")]
    results = []
    for i in (ids[0], ids[-1]):
        pool.write(i, m, h)
        out = torch.zeros((25, 4096), device="cuda")
        torch.cuda.synchronize()
        pkg.gdn_tree_forward(backend, pool, [i], [25], tree, *x, *w, out)
        pkg.gdn_tree_commit(backend, [(pool, i, 24)])
        results.append([out.cpu().numpy(), *pool.read(i)])
    for first, last in zip(*results):
        assert np.array_equal(first, last)
    assert not np.array_equal(results[0][1], m)
    pool.destroy()
