"""attention_tree_forward against the formula in 64 bits.

Row r attends to the context, its ancestors and itself.  The cache holds keys
and values in bf16: the appended ones are read back and held to the formula's
by half a bf16 step (2^-8) and the f32 error of norm and RoPE, and the outputs
are compared on the cache as it is, so that a key that rounds the other way
does not widen the bound of the outputs.

Bound of an output, with A = sum p |v| / sum p and S the largest sum |q k| /
sqrt(D) of a visible key: q carries 32 roundings of 2^-24 (norm, RoPE, scale)
and its parts 2^-24 (f32 out) or 2^-16; a score's sum D more: dS; a weight is
off by 2 dS (its own and the sum's) and by its parts and the exponential, together
2^-22 (f32 out: 2^-24 and a unit in the last place, 2^-23) or 2^-8; n weights are
summed.
"""
import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")


def random_tree(rng, rows, depth=8):
    parents, depths = [], []
    for i in range(rows):
        p = -1 if i == 0 or rng.random() < 0.2 else int(rng.integers(max(0, i - 9), i))
        if p >= 0 and depths[p] + 1 >= depth:
            p = parents[p]
        parents.append(p)
        depths.append(0 if p < 0 else depths[p] + 1)
    return parents, depths


def ancestors(parents, r):
    path = []
    while r >= 0:
        path.append(r)
        r = parents[r]
    return path[::-1]


def rope64(x, angle, rot):
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    left, right = x[..., :rot // 2], x[..., rot // 2:rot]
    return np.concatenate([left * c - right * s, right * c + left * s, x[..., rot:]], -1)


class Case:
    def __init__(self, backend, seed, heads, kvh, dim, rot, trees, contexts, *, page=64, norm=True,
                 gated=False, bf16=False, out16=False, theta=1e6, scattered=False, scale=1.0,
                 mrope=(0, 0, 0), device=True):
        self.__dict__.update(heads=heads, kvh=kvh, dim=dim, rot=rot, trees=trees, contexts=contexts,
                             norm=norm, gated=gated, bf16=bf16, out16=out16, theta=theta,
                             mrope=mrope, backend=backend)
        rng = np.random.default_rng(seed)
        rows = sum(len(t) for t in trees)
        self.rows = rows
        most = max(c + len(t) for c, t in zip(contexts, trees))
        self.pool = pkg.KvCache(backend, kvh, dim, page, len(trees) * (most // page + 2) + 4,
                                most + 3, len(trees) + 2, page_order_seed=seed + 1 if scattered else 0)
        self.ids = [self.pool.open() for _ in trees]
        self.cached = []
        for i, c in zip(self.ids, contexts):
            k, v = (torch.from_numpy(rng.standard_normal((c, kvh * dim)).astype(np.float32)).bfloat16()
                    for _ in range(2))
            if c:
                self.pool.append(i, k.cuda(), v.cuda())
            self.cached.append((k.double().numpy(), v.double().numpy()))
        dtype = torch.bfloat16 if bf16 else torch.float32
        hs = dim * (2 if gated else 1)

        def tensor(*shape):
            return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * scale).to(dtype)

        self.q, self.k, self.v = tensor(rows, heads * hs), tensor(rows, kvh * dim), tensor(rows, kvh * dim)
        self.gains = [torch.from_numpy((0.0 if gated else 1.0) +
                                       0.1 * rng.standard_normal(dim)).float() for _ in range(2)]
        pos = []
        for c, t in zip(contexts, trees):
            for r in range(len(t)):
                p = c + len(ancestors(t, r)) - 1
                pos.append([p, p + (3 if any(mrope) else 0), p + (7 if any(mrope) else 0)])
        self.pos = torch.tensor(pos, dtype=torch.int32)
        self.device = device

    def run(self, asynchronous=False):
        out = torch.full((self.rows, self.heads * self.dim), math.nan,
                         dtype=torch.bfloat16 if self.out16 else torch.float32)
        put = (lambda t: t.cuda()) if self.device else (lambda t: t.numpy())
        args = [put(t) for t in (self.q, self.k, self.v, self.pos, out)]
        gains = [put(g) for g in self.gains] if self.norm else [None, None]
        pkg.attention_tree_forward(
            self.backend, self.pool, self.ids, [len(t) for t in self.trees],
            [p for t in self.trees for p in t], *args, heads=self.heads, kv_heads=self.kvh,
            head_dim=self.dim, rotary_dim=self.rot, rope_theta=self.theta, q_norm=gains[0],
            k_norm=gains[1], gated=self.gated, norm_offset=self.gated, mrope_section=self.mrope,
            asynchronous=asynchronous)
        if asynchronous:
            self.backend.synchronize()
        return args[-1].cpu() if self.device else torch.from_numpy(args[-1])

    def prepared(self):
        """q and k after norm and RoPE, and the sums of magnitudes behind them."""
        q = self.q.double().numpy().reshape(self.rows, self.heads, -1)
        k = self.k.double().numpy().reshape(self.rows, self.kvh, self.dim)
        gate = q[..., self.dim:] if self.gated else None
        q = q[..., :self.dim]
        if self.norm:
            add = 1.0 if self.gated else 0.0
            q, k = (x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))
                    * (g.double().numpy() + add) for x, g in zip((q, k), self.gains))
        half = self.rot // 2
        power = np.array([math.pow(self.theta, 2 * i / self.rot) for i in range(half)], np.float32)
        axis = np.zeros(half, int)
        if any(self.mrope):
            i = np.arange(half)
            axis[(i % 3 == 1) & (i < 3 * self.mrope[1])] = 1
            axis[(i % 3 == 2) & (i < 3 * self.mrope[2])] = 2
        angle = (self.pos.numpy()[:, axis].astype(np.float32) / power).astype(np.float64)
        return rope64(q, angle, self.rot), rope64(k, angle, self.rot), gate

    def check(self, got):
        q, k, gate = self.prepared()
        at = 0
        worst = 0.0
        for i, (c, tree) in enumerate(zip(self.contexts, self.trees)):
            n = len(tree)
            assert self.pool.len(self.ids[i]) == c + n
            keys, values = (x.astype(np.float64) for x in self.pool.read(self.ids[i]))
            assert np.array_equal(keys[:c], self.cached[i][0])
            assert np.array_equal(values[:c], self.cached[i][1])
            new = k[at:at + n].reshape(n, -1)
            size = np.sqrt((new.reshape(n, self.kvh, -1) ** 2).max(-1, keepdims=True))
            slack = 2.0 ** -8 * np.abs(new) + np.broadcast_to(
                32 * 2.0 ** -24 * 2 * size, (n, self.kvh, self.dim)).reshape(n, -1)
            assert np.all(np.abs(keys[c:] - new) <= slack)
            assert np.array_equal(values[c:], self.v[at:at + n].to(torch.bfloat16).double().numpy())
            keys, values = keys.reshape(c + n, self.kvh, -1), values.reshape(c + n, self.kvh, -1)
            for r in range(n):
                see = list(range(c)) + [c + a for a in ancestors(tree, r)]
                for h in range(self.heads):
                    kk, vv = keys[see, h // (self.heads // self.kvh)], values[see, h // (self.heads // self.kvh)]
                    s = kk @ q[at + r, h] / math.sqrt(self.dim)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    want, mag = p @ vv, p @ np.abs(vv)
                    big = (np.abs(kk) @ np.abs(q[at + r, h])).max() / math.sqrt(self.dim)
                    ds = big * ((32 + self.dim) * 2.0 ** -24 + (2.0 ** -16 if self.out16 else 2.0 ** -24))
                    tol = mag * (2 * ds + (2.0 ** -8 if self.out16 else 2.0 ** -22) +
                                 (len(see) + 64) * 2.0 ** -24)
                    if gate is not None:
                        g = 1 / (1 + np.exp(-gate[at + r, h]))
                        want, tol = want * g, tol * g + np.abs(want * g) * 8 * 2.0 ** -24
                    if self.out16:
                        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
                    err = np.abs(got[at + r, h * self.dim:(h + 1) * self.dim].double().numpy() - want)
                    worst = max(worst, float((err / (tol + 1e-30)).max()))
            at += n
        assert worst <= 1.0, f"error {worst:.2f} times the bound"


SHAPES = {  # heads, KV heads, head_dim, rotary_dim
    "64": (14, 2, 64, 64),
    "128": (8, 2, 128, 128),
    "256": (8, 1, 256, 64),
    "80": (6, 2, 80, 40),
    "mha": (3, 3, 128, 64),
    "group12": (12, 1, 64, 32),
    "512": (2, 1, 512, 512),
    "18": (4, 2, 18, 6),
}


@pytest.mark.parametrize("out16", [False, True])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_tree(backend, shape, out16):
    heads, kvh, dim, rot = SHAPES[shape]
    rng = np.random.default_rng(11)
    trees = [random_tree(rng, n)[0] for n in (1, 7, 20)]
    case = Case(backend, 5, heads, kvh, dim, rot, trees, [0, 63, 201], bf16=out16, out16=out16)
    case.check(case.run())
    case.pool.destroy()


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 64, 65, 96, 127, 128])
@pytest.mark.parametrize("context", [0, 1, 31, 100, 129])
def test_rows_and_contexts(backend, rows, context):
    """The rows' mask at every place of a tile; a context of none."""
    tree = random_tree(np.random.default_rng(rows), rows, 40)[0]
    case = Case(backend, rows, 4, 2, 128, 128, [tree], [context], page=16, scattered=True)
    case.check(case.run())
    case.pool.destroy()


@pytest.mark.parametrize("dim,heads,kvh", [(64, 8, 1), (128, 8, 1), (256, 4, 1)])
@pytest.mark.parametrize("context", [4500, 8191])
def test_partitions(backend, dim, heads, kvh, context):
    """Contexts cut over many workgroups and joined."""
    rng = np.random.default_rng(3)
    trees = [random_tree(rng, n)[0] for n in (5, 17)]
    case = Case(backend, 9, heads, kvh, dim, dim, trees, [context, 1000], page=16, scattered=True,
                norm=False, gated=True, bf16=True)
    case.check(case.run())
    case.pool.destroy()


@pytest.mark.parametrize("gated,norm,mrope", [(True, True, (11, 11, 10)), (False, False, (0, 0, 0)),
                                              (True, False, (0, 0, 0))])
@pytest.mark.parametrize("device", [True, False])
def test_forms(backend, gated, norm, mrope, device):
    tree = random_tree(np.random.default_rng(1), 13)[0]
    case = Case(backend, 3, 4, 2, 64, 64, [tree], [130], gated=gated, norm=norm, mrope=mrope,
                device=device)
    case.check(case.run(asynchronous=device))
    case.pool.destroy()


def test_many_sequences(backend):
    """More sequences and rows than one launch takes."""
    rng = np.random.default_rng(2)
    trees = [random_tree(rng, int(rng.integers(1, 60)))[0] for _ in range(45)]
    contexts = [int(rng.integers(0, 90)) for _ in trees]
    case = Case(backend, 7, 2, 1, 64, 64, trees, contexts, page=16)
    case.check(case.run())
    case.pool.destroy()


def test_large_scores(backend):
    """Scores of several hundred: the maximum moves, weights fall to zero."""
    tree = random_tree(np.random.default_rng(4), 9)[0]
    case = Case(backend, 4, 4, 2, 128, 128, [tree], [700], norm=False, scale=20.0)
    case.check(case.run())
    case.pool.destroy()


def test_chain_is_attention_forward(backend):
    """A chain gives attention_forward's rows, within that call's fp16 tolerance."""
    case = Case(backend, 6, 8, 2, 128, 128, [[-1, 0, 1, 2, 3]], [500])
    got = case.run()
    case.check(got)
    case.pool.truncate(case.ids[0], 500)
    out = torch.zeros((5, 8 * 128), device="cuda")
    pkg.attention_forward(backend, case.pool, case.ids, [5], case.q.cuda(), case.k.cuda(),
                          case.v.cuda(), case.pos.cuda(), out, heads=8, kv_heads=2, head_dim=128,
                          rotary_dim=128, rope_theta=1e6, q_norm=case.gains[0].cuda(),
                          k_norm=case.gains[1].cuda())
    assert torch.all((out.cpu() - got).abs() <= 2e-3 + 1e-2 * got.abs())
    case.pool.destroy()


def test_shared_pages_are_copied(backend):
    """A fork's tree leaves the other's partly filled page as it was."""
    tree = random_tree(np.random.default_rng(8), 12)[0]
    case = Case(backend, 2, 4, 2, 64, 64, [tree], [70])
    fork = case.pool.fork(case.ids[0])
    before = case.pool.read(fork)
    case.check(case.run())
    after = case.pool.read(fork)
    assert all(np.array_equal(x, y) for x, y in zip(before, after))
    case.pool.destroy()


def test_non_finite_rows_change_nothing(backend):
    case = Case(backend, 2, 4, 2, 64, 64, [[-1, 0, 0]], [70])
    case.v[1, 5] = math.inf
    with pytest.raises(pkg.PluginError, match="non-finite"):
        case.run()
    assert case.pool.len(case.ids[0]) == 70
    case.v[1, 5] = 0.0
    case.check(case.run())
    case.pool.destroy()


def test_repeats_are_bit_equal(backend):
    rng = np.random.default_rng(5)
    case = Case(backend, 1, 8, 1, 128, 128, [random_tree(rng, 40)[0], random_tree(rng, 3)[0]],
                [3000, 40], bf16=True)
    outs = []
    for _ in range(3):
        outs.append(case.run())
        for i, c in zip(case.ids, case.contexts):
            case.pool.truncate(i, c)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    case.pool.destroy()


@pytest.mark.parametrize("change,text", [
    (dict(parents=[0, 0, 1]), "parent"),
    (dict(parents=[-1, 2, 1]), "parent"),
    (dict(parents=[-1, -2, 1]), "parent"),
    (dict(ids=[0, 0], rows=[1, 2], parents=[-1, -1, 0]), "twice"),
    (dict(rows=[0], parents=[]), "empty"),
    (dict(ids=[9]), "not open"),
    (dict(rotary=65), "RoPE"),
])
def test_refusals(backend, change, text):
    case = Case(backend, 2, 4, 2, 64, 64, [[-1, 0, 1]], [70])
    out = torch.zeros((3, 4 * 64), device="cuda")
    with pytest.raises(pkg.PluginError, match=text):
        pkg.attention_tree_forward(backend, case.pool, change.get("ids", [0]), change.get("rows", [3]),
                                   change.get("parents", [-1, 0, 1]), case.q.cuda(), case.k.cuda(),
                                   case.v.cuda(), case.pos.cuda(), out, heads=4, kv_heads=2,
                                   head_dim=64, rotary_dim=change.get("rotary", 64), rope_theta=1e6)
    assert case.pool.len(0) == 70
    case.pool.destroy()


def test_refuses_too_many_rows(backend):
    case = Case(backend, 2, 4, 2, 64, 64, [list(range(-1, 127))], [0])
    big = torch.zeros((129, 4 * 64), device="cuda")
    pos = torch.zeros((129, 3), dtype=torch.int32, device="cuda")
    with pytest.raises(pkg.PluginError, match="MAX_TREE_ROWS"):
        pkg.attention_tree_forward(backend, case.pool, [0], [129], list(range(-1, 128)), big,
                                   big[:, :128].contiguous(), big[:, :128].contiguous(), pos, big,
                                   heads=4, kv_heads=2, head_dim=64, rotary_dim=64, rope_theta=1e6)
    case.check(case.run())
    case.pool.destroy()
