"""kv_compact and kv_gather against lists of rows on the host: copies, so every
comparison is for equality."""
import ctypes as C
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
pkg = importlib.import_module("safetyraise-lmengine_amd")


def rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    return torch.from_numpy(x).bfloat16().float().numpy()


class Model:
    """A pool and, per open sequence, the rows it must hold."""

    def __init__(self, backend, rng, kvh=2, dim=64, page=16, pages=200, slots=12, seed=0):
        self.backend, self.rng, self.width = backend, rng, kvh * dim
        self.pool = pkg.KvCache(backend, kvh, dim, page, pages, 4096, slots, page_order_seed=seed)
        self.held = {}

    def new(self, n):
        s = self.pool.open()
        k, v = (rows(self.rng, n, self.width) for _ in range(2))
        if n:
            self.pool.append(s, k, v)
        self.held[s] = (k, v)
        return s

    def append(self, s, n):
        k, v = (rows(self.rng, n, self.width) for _ in range(2))
        self.pool.append(s, k, v)
        self.held[s] = tuple(np.concatenate(x) for x in zip(self.held[s], (k, v)))

    def fork(self, s):
        f = self.pool.fork(s)
        self.held[f] = self.held[s]
        return f

    def kept(self, source, start, tokens):
        at = list(range(start)) + [start + t for t in tokens]
        return tuple(x[at] for x in self.held[source])

    def check(self):
        for s, (k, v) in self.held.items():
            assert self.pool.len(s) == len(k)
            got = self.pool.read(s)
            assert np.array_equal(got[0], k) and np.array_equal(got[1], v), f"sequence {s}"


def compact(backend, entries, asynchronous=False):
    """entries: (model, source, target, start, tokens)"""
    after = [(m, target, m.kept(source, start, tokens)) for m, source, target, start, tokens in entries]
    pkg.kv_compact(backend, [(m.pool, *rest) for m, *rest in entries], asynchronous=asynchronous)
    for m, target, held in after:
        m.held[target] = held


@pytest.mark.parametrize("dim", [64, 128, 40, 18, 7])
@pytest.mark.parametrize("page", [16, 64])
def test_commit_in_place(backend, dim, page):
    """A path of a few drafts behind contexts that end anywhere in a page."""
    rng = np.random.default_rng(dim)
    m = Model(backend, rng, 3, dim, page)
    for context in (0, 1, 15, 16, 17, 63, 64, 100):
        s = m.new(context + 20)
        compact(backend, [(m, s, s, context, sorted(rng.choice(20, 5, replace=False).tolist()))])
    m.check()
    for s in list(m.held):
        m.append(s, 7)  # appends go on behind the kept tokens
    m.check()
    m.pool.destroy()


@pytest.mark.parametrize("dim", [257, 300, 511, 512])
def test_wide_rows(backend, dim):
    """Rows of more units than a workgroup has threads."""
    rng = np.random.default_rng(dim)
    m = Model(backend, rng, 2, dim, 16)
    s, b, c = m.new(60), m.new(90), m.new(0)
    compact(backend, [(m, s, s, 33, [1, 2, 7, 20]), (m, b, c, 10, list(range(0, 80, 3)))])
    m.check()
    k, v = (np.zeros((39, m.width), np.float32) for _ in range(2))
    pkg.kv_gather(backend, [(m.pool, c, 5, [0, 7, 3]), (m.pool, s, 0, 36)], k, v)
    at = [5, 12, 8]
    for got, c_rows, s_rows in ((k, m.held[c][0], m.held[s][0]), (v, m.held[c][1], m.held[s][1])):
        assert np.array_equal(got, np.concatenate([c_rows[at], s_rows[:36]]))
    m.pool.destroy()


def test_pages_given_up_are_still_read(backend):
    """A page that one entry gives up is no free page to the entries behind it: the
    call's copies still read it."""
    rng = np.random.default_rng(11)
    for page in (16, 64):
        m = Model(backend, rng, 2, 64, page, pages=40)
        a, b, c = m.new(5 * page - 1), m.new(4 * page), m.new(0)
        tokens = [2 * page + 3, 3 * page + 1, 4 * page + 2]
        compact(backend, [(m, a, a, page + 2, [t - page - 2 for t in tokens]),
                          (m, b, c, 3, list(range(0, 4 * page - 3, 2)))])
        m.check()
        m.pool.destroy()


@pytest.mark.parametrize("tokens", [[], [0], [19], list(range(20)), list(range(5)), list(range(16, 20)),
                                    list(range(4, 20))])
def test_edges(backend, tokens):
    """Nothing kept, everything, prefixes, suffixes: links and truncations."""
    for start in (0, 12, 16, 32):
        m = Model(backend, np.random.default_rng(1))
        s, t = m.new(start + 20), m.new(5)
        compact(backend, [(m, s, t, start, tokens)])
        m.check()
        compact(backend, [(m, s, s, start, tokens)])
        m.check()
        m.append(s, 40)
        m.append(t, 3)
        m.check()
        m.pool.destroy()


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("tight", [False, True])
def test_long(backend, into, tight):
    """Thousands of tokens: to free pages, or in place when there are none."""
    rng = np.random.default_rng(7)
    m = Model(backend, rng, 2, 128, 16, pages=130 if tight else 600)
    if into and tight:
        s = m.new(1000)
    else:
        s = m.new(2000)
    n = m.pool.len(s)
    t = m.new(3) if into else s
    keep = sorted(rng.choice(n - 37, n // 2, replace=False).tolist())
    keep = [x for x in keep if not 300 <= x < 400] + list(range(n - 37, n - 20))
    compact(backend, [(m, s, t, 37, sorted(set(x for x in keep if x < n - 37)))], asynchronous=True)
    m.check()
    m.append(t, 30)
    m.check()
    m.pool.destroy()


def test_shared_pages_stay(backend):
    """Forks keep their rows whatever happens to the others' pages."""
    rng = np.random.default_rng(3)
    m = Model(backend, rng)
    s = m.new(100)
    a, b = m.fork(s), m.fork(s)
    m.append(a, 9)
    compact(backend, [(m, a, a, 90, [1, 4, 18])])
    m.check()
    compact(backend, [(m, b, b, 0, list(range(16, 48)) + [50, 99])])
    m.check()
    m.pool.truncate(s, 20)
    m.held[s] = tuple(x[:20] for x in m.held[s])
    compact(backend, [(m, b, s, 3, [0, 2, 9])])
    m.check()
    m.pool.destroy()


def test_random_operations(backend):
    """Hundreds of calls over forks, appends, truncations, closes and compactions."""
    rng = np.random.default_rng(11)
    m = Model(backend, rng, 1, 64, 16, pages=150, slots=10, seed=5)
    m.new(40)
    for step in range(400):
        s = int(rng.choice(list(m.held)))
        n = len(m.held[s][0])
        op = rng.integers(0, 8)
        try:
            if op == 0 and len(m.held) < 9:
                m.new(int(rng.integers(0, 80)))
            elif op == 1 and len(m.held) < 9:
                m.fork(s)
            elif op == 2:
                m.append(s, int(rng.integers(1, 60)))
            elif op == 3 and len(m.held) > 2:
                m.pool.close(s)
                del m.held[s]
            elif op == 4:
                cut = int(rng.integers(0, n + 1))
                m.pool.truncate(s, cut)
                m.held[s] = tuple(x[:cut] for x in m.held[s])
            else:
                start = int(rng.integers(0, n + 1))
                keep = np.flatnonzero(rng.random(n - start) < rng.choice([0.1, 0.5, 0.9, 1.0])).tolist()
                t = s if rng.random() < 0.6 else int(rng.choice(list(m.held)))
                compact(backend, [(m, s, t, start, keep)], asynchronous=True)
        except pkg.PluginError as e:
            assert e.status == 4, e  # the pool is full: nothing changed
        if step % 10 == 9:
            m.check()
    m.check()
    m.pool.destroy()


def test_many_pools(backend):
    """Layers of several geometries and sequences in one call, long and short."""
    rng = np.random.default_rng(2)
    models = [Model(backend, rng, kvh, dim, page, pages=120, seed=i)
              for i, (kvh, dim, page) in enumerate([(2, 64, 16), (1, 128, 64), (3, 36, 16)] * 6)]
    entries = []
    for m in models:
        a, b, c = m.new(60), m.new(300), m.new(0)
        entries += [(m, a, a, 40, [2, 5, 11]), (m, b, c, 10, sorted(rng.choice(290, 100, replace=False).tolist()))]
    compact(backend, entries, asynchronous=True)
    for m in models:
        m.check()
        m.pool.destroy()


def test_commit_follows_a_tree(backend):
    """attention_tree_forward, kv_compact, attention_forward: the committed rows are
    the path's."""
    rng = np.random.default_rng(4)
    m = Model(backend, rng, 2, 64, 16)
    s = m.new(50)
    q = torch.randn(6, 4 * 64, device="cuda")
    k, v = (torch.randn(6, 2 * 64, device="cuda") for _ in range(2))
    out = torch.zeros_like(q)
    parents = [-1, -1, 1, 1, 3, 0]
    pos = torch.tensor([[50 + d] * 3 for d in (0, 0, 1, 1, 2, 1)], dtype=torch.int32, device="cuda")
    kw = dict(heads=4, kv_heads=2, head_dim=64, rotary_dim=64, rope_theta=1e6)
    pkg.attention_tree_forward(backend, m.pool, [s], [6], parents, q, k, v, pos, out, **kw)
    pkg.kv_compact(backend, [(m.pool, s, s, 50, [1, 3, 4])], asynchronous=True)
    chain = m.new(0)
    pkg.kv_compact(backend, [(m.pool, s, chain, 50, [])])
    again = torch.zeros((3, 4 * 64), device="cuda")
    path = [1, 3, 4]
    pkg.attention_tree_forward(backend, m.pool, [chain], [3], [-1, 0, 1], q[path], k[path], v[path],
                               pos[path], again, **kw)
    a, b = m.pool.read(s), m.pool.read(chain)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    # (other key orders in the sums: f32 roundings of 55 terms of about 1)
    assert torch.all((again - out[path]).abs() <= 55 * 2.0 ** -16)
    m.pool.destroy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 40, 18])
def test_gather(backend, dtype, dim):
    rng = np.random.default_rng(6)
    m = Model(backend, rng, 3, dim, 16, seed=3)
    other = Model(backend, rng, 3, dim, 64)
    a, b, c = m.new(100), m.new(33), other.new(200)
    for count in (1, 40, 3000):
        pick = rng.integers(0, 90, count).tolist()  # any order, repeats
        reads = [(m, a, 10, pick), (m, b, 0, 33), (m, b, 33, 0), (other, c, 150, 50), (other, c, 0, [199])]
        total = count + 33 + 50 + 1
        k, v = (torch.full((total, m.width), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        pkg.kv_gather(backend, [(x.pool, s, start, t) for x, s, start, t in reads], k, v, asynchronous=True)
        backend.synchronize()
        for got, which in ((k, 0), (v, 1)):
            want = np.concatenate([x.held[s][which][[start + j for j in (range(t) if isinstance(t, int) else t)]]
                                   for x, s, start, t in reads])
            assert np.array_equal(got.float().cpu().numpy(), want)
    host = [np.zeros((33, m.width), np.float32) for _ in range(2)]
    pkg.kv_gather(backend, [(m.pool, b, 0, 33)], *host)
    assert np.array_equal(host[0], m.held[b][0]) and np.array_equal(host[1], m.held[b][1])
    m.pool.destroy()
    other.pool.destroy()


def test_refusals(backend):
    rng = np.random.default_rng(1)
    m = Model(backend, rng, pages=12)
    a, b = m.new(50), m.new(20)

    def refused(text, *entries):
        with pytest.raises(pkg.PluginError, match=text):
            pkg.kv_compact(backend, [(m.pool, *e) for e in entries])
        m.check()

    refused("ascend", (a, a, 0, [3, 3]))
    refused("ascend", (a, a, 0, [4, 3]))
    refused("ascend", (a, a, 40, [10]))
    refused("out of range", (a, a, 51, []))
    refused("not open", (a, 7, 0, [1]))
    refused("not open", (9, a, 0, [1]))
    refused("another entry", (a, a, 0, [1]), (a, b, 0, [1]))
    refused("another entry", (a, b, 0, [1]), (b, b, 0, [1]))
    refused("another entry", (a, b, 0, [1]), (a, b, 0, [2]))
    f = m.fork(a)
    g = m.new(48)
    refused("exhausted", (f, f, 0, [x for x in range(50) if x != 1]), (g, g, 0, list(range(1, 48))),
            (a, b, 0, [x for x in range(50) if x != 2]))
    k = torch.zeros((4, m.width), device="cuda")
    for bad in ((a, 0, [50]), (a, 51, 0), (a, 49, 2)):
        with pytest.raises(pkg.PluginError, match="out of range"):
            pkg.kv_gather(backend, [(m.pool, *bad)], k, k.clone())
    m.pool.destroy()


@pytest.mark.parametrize("token", [50, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 1, 2 ** 32 - 1])
@pytest.mark.parametrize("at", [0, 7, 20])
def test_tokens_out_of_range(backend, token, at):
    """One token too large, anywhere in a list, in every place of a vector."""
    m = Model(backend, np.random.default_rng(1))
    a, b = m.new(50), m.new(20)
    good = list(range(20))
    k, v = (np.zeros((21, m.width), np.float32) for _ in range(2))
    with pytest.raises(pkg.PluginError, match="out of range"):
        pkg.kv_gather(backend, [(m.pool, a, 0, good[:at] + [token] + good[at:])], k, v)
    for tokens in (good[:at] + [token], good[:at] + [token] + [x + 21 for x in good[at:]], [5, 5], [9, 8, 10]):
        with pytest.raises(pkg.PluginError, match="ascend strictly"):
            pkg.kv_compact(backend, [(m.pool, a, b, 0, tokens)])
        m.check()
    # a list that two entries share: within one sequence, beyond the other
    shared = (C.c_uint32 * 21)(*range(21))
    k, v = (np.zeros((42, m.width), np.float32) for _ in range(2))
    for order, status in (((a, b), 1), ((b, a), 1), ((a, a), 0)):
        entries = (pkg.plugin.KvRows * 2)()
        for e, sequence in zip(entries, order):
            e.kv, e.sequence, e.count, e.tokens = m.pool.handle, sequence, 21, shared
        assert status == backend.lib.safetyraise_kernel_kv_gather(
            backend.context, entries, 2, k.ctypes.data, v.ctypes.data, 0)
    assert np.array_equal(k, np.concatenate([m.held[a][0][:21]] * 2))
    m.pool.destroy()


def test_tensors_of_another_stream(backend):
    """Calls on a stream of the caller's, between its own work."""
    rng = np.random.default_rng(9)
    m = Model(backend, rng)
    s = m.new(64)
    stream = torch.cuda.Stream()
    backend.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            k, v = (torch.randn(20, m.width, device="cuda").bfloat16() for _ in range(2))
            m.pool.append(s, k, v, flags=pkg.ASYNC)
            compact_tokens = [0, 3, 19]
            pkg.kv_compact(backend, [(m.pool, s, s, 64, compact_tokens)], asynchronous=True)
            gk, gv = (torch.empty(3, m.width, device="cuda", dtype=torch.bfloat16) for _ in range(2))
            pkg.kv_gather(backend, [(m.pool, s, 64, 3)], gk, gv, asynchronous=True)
            gk2 = gk * 2
        stream.synchronize()
        assert torch.equal(gk, k[compact_tokens]) and torch.equal(gv, v[compact_tokens])
        assert torch.equal(gk2, k[compact_tokens] * 2)
    finally:
        backend.set_stream(None)
    m.pool.destroy()
