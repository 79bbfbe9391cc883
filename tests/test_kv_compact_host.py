"""kv_compact and kv_gather on the library's host code, the copies done on the host in any
order that the launches allow (host_library.cpp): contents, page lists, reference counts
and free lists after every call."""
import ctypes as C
import importlib

import numpy as np
import pytest

from host_library import host, host_path  # noqa: F401

pkg = importlib.import_module("safetyraise-lmengine_amd")
KVH, DIM = 1, 2


class Model:
    """A pool and, per open sequence, the tokens that it must hold (a token's rows are
    numbers of its own)."""
    count = 0

    def __init__(self, backend, page=16, pages=64, slots=12):
        self.backend, self.page = backend, page
        self.pool = pkg.KvCache(backend, KVH, DIM, page, pages, 4096, slots)
        self.held = {}

    def rows(self, n):
        at = np.arange(Model.count, Model.count + n, dtype=np.float32) % 65536
        Model.count += n
        k = np.stack([at // 256, at % 256], 1).astype(np.float32)  # (exact in bf16: 8 bits each)
        return k, -k

    def new(self, n):
        s = self.pool.open()
        self.held[s] = [np.zeros((0, KVH * DIM), np.float32)] * 2
        if n:
            self.append(s, n)
        return s

    def append(self, s, n):
        k, v = self.rows(n)
        self.pool.append(s, k, v)
        self.held[s] = [np.concatenate(x) for x in zip(self.held[s], (k, v))]

    def fork(self, s):
        f = self.pool.fork(s)
        self.held[f] = self.held[s]
        return f

    def close(self, s):
        self.pool.close(s)
        del self.held[s]

    def kept(self, source, start, tokens):
        at = list(range(start)) + [start + t for t in tokens]
        return [x[at] for x in self.held[source]]

    @property
    def free(self):
        return self.backend.test.test_free_pages(self.pool.handle)

    def check(self):
        wrong = self.backend.test.test_pool(self.pool.handle)
        assert wrong == 0, ["", "reference counts", "free list", "page table", "pages"][wrong]
        for s, (k, v) in self.held.items():
            assert self.pool.len(s) == len(k)
            got = self.pool.read(s)
            assert np.array_equal(got[0], k) and np.array_equal(got[1], v), f"sequence {s}"


def call(backend, entries):
    """entries: (model, source, target, start, tokens), tokens a ctypes array or a list;
    arrays are passed as they are, so that entries can share one.  The status."""
    keeps = (pkg.plugin.KvKeep * len(entries))()
    held = []
    for e, (m, source, target, start, tokens) in zip(keeps, entries):
        if not isinstance(tokens, C.Array):
            tokens = (C.c_uint32 * max(1, len(tokens)))(*tokens) if len(tokens) else None
        held.append(tokens)
        e.kv, e.source, e.target, e.start = m.pool.handle, source, target, start
        e.count = len(tokens) if tokens is not None else 0
        if tokens is not None:
            e.tokens = tokens
    after = [(m, target, m.kept(source, start, list(tokens) if tokens is not None else []))
             for (m, source, target, start, _), tokens in zip(entries, held)]
    status = backend.lib.safetyraise_kernel_kv_compact(backend.context, keeps, len(entries), 0)
    if status == 0:
        for m, target, rows in after:
            m.held[target] = rows
    return status


def shared(tokens):
    return (C.c_uint32 * len(tokens))(*tokens)


def test_random_calls(host):  # noqa: F811
    """Calls of several entries over several pools, token lists shared between them."""
    rng = np.random.default_rng(1)
    host.test.test_seed(7)
    models = [Model(host, page, pages) for page, pages in ((16, 22), (16, 60), (32, 12))]
    for m in models:
        for n in (40, 100, 3):
            m.new(n)
    full = several = 0
    for step in range(12000):
        m = models[int(rng.integers(len(models)))]
        s = int(rng.choice(list(m.held)))
        n = len(m.held[s][0])
        op = int(rng.integers(0, 10))
        try:
            if op == 0 and len(m.held) < 9:
                m.new(int(rng.integers(0, 80)))
            elif op == 1 and len(m.held) < 9:
                m.fork(s)
            elif op in (2, 3, 4):
                if rng.random() < 0.1:  # pages past its length, that hold nothing
                    host.test.test_fail(b"kv_scatter", 0)
                    with pytest.raises(pkg.PluginError):
                        m.pool.append(s, *m.rows(int(rng.integers(1, 90))))
                    host.test.test_fail(b"", 0)
                else:
                    m.append(s, int(rng.integers(1, 90)))
            elif op == 5 and len(m.held) > 4:
                m.close(s)
            elif op == 6 and rng.random() < 0.3:
                cut = int(rng.integers(0, n + 1))
                m.pool.truncate(s, cut)
                m.held[s] = [x[:cut] for x in m.held[s]]
        except pkg.PluginError as e:
            assert e.status == 4, e
        if op < 8:
            continue
        # entries that share a list where it fits
        start = int(rng.integers(0, n + 1))
        tokens = shared(np.flatnonzero(rng.random(n - start) < rng.choice([0.3, 0.9, 0.97, 1.0])).tolist())
        if len(tokens) == 0 and rng.random() < 0.95:
            continue
        entries, used = [], set()
        for m in models:
            for s in rng.permutation(list(m.held)):
                s = int(s)
                n = len(m.held[s][0])
                fits = start <= n and (len(tokens) == 0 or start + tokens[-1] < n)
                if not fits or (m, s) in used or rng.random() < 0.7:
                    continue
                others = [t for t in m.held if (m, t) not in used and t != s]
                t = s if rng.random() < 0.6 or not others else int(rng.choice(others))
                used |= {(m, s), (m, t)}
                entries.append((m, s, t, start, tokens if len(tokens) else []))
        if entries:
            status = call(host, entries)
            assert status in (0, 4)
            full += status == 4
            several += status == 0 and len(entries) > 3
        for m in models:
            m.check()
    assert full > 30 and several > 300
    for m in models:
        m.pool.destroy()


def layers(backend, n=3, tokens=700, **change):
    """Pools with a sequence 0 of `tokens` tokens; change: per layer, other arguments."""
    models = [Model(backend, **dict(dict(page=16, pages=160), **change.get(f"layer{i}", {}))) for i in range(n)]
    for m in models:
        m.new(tokens)
    return models


KEPT = [t for t in range(0, 600) if t % 7 not in (2, 5)]  # (long: to free pages where there are some)
PATH = [1, 2, 5, 9]
LISTS = {"long": KEPT, "path": PATH}


@pytest.mark.parametrize("which", list(LISTS))
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 0, 2)])
@pytest.mark.parametrize("odd", ["none", "fork", "page", "start", "target", "tight"])
def test_layers_share_a_list(host, odd, order, which):  # noqa: F811
    """Layers with one token array, as an engine passes it: plans are shared where they may
    be.  One layer differs in one thing."""
    tokens = shared(LISTS[which])
    change = {"page": dict(page=64, pages=40), "tight": dict(pages=46)}.get(odd, {})
    models = layers(host, layer1=change)
    odd_one = models[1]
    start = {m: 40 for m in models}
    target = {m: 0 for m in models}
    if odd == "fork":
        odd_one.fork(0)  # its pages are shared
    if odd == "start":
        start[odd_one] = 41
    if odd == "target":
        target[odd_one] = odd_one.new(5)
    entries = [(models[i], 0, target[models[i]], start[models[i]], tokens) for i in order]
    assert call(host, entries) == 0
    for m in models:
        m.check()
    for m in models:  # the sequences go on
        m.append(target[m], 20)
        m.check()
        m.pool.destroy()


def test_sequences_share_a_list(host):  # noqa: F811
    """Sequences of one pool with one token array, some forked, in place and into others,
    the free pages used up on the way."""
    for pages in (230, 130, 112, 108):
        m = Model(host, pages=pages)
        tokens = shared(KEPT)
        a, b, c = m.new(641), m.new(650), m.new(30)
        f = m.fork(c)
        entries = [(m, a, a, 40, tokens), (m, b, c, 40, tokens)]
        status = call(host, entries)
        assert status in (0, 4)
        m.check()
        assert f in m.held and m.pool.len(f) == 30
        if status == 4:
            assert call(host, entries[:1]) == 0
            m.check()
        m.pool.destroy()


def test_gather_shares_a_list(host):  # noqa: F811
    m, other = Model(host, 16), Model(host, 64)
    a, b = m.new(300), other.new(500)
    tokens = shared([7, 3, 3, 250, 0])
    reads = (pkg.plugin.KvRows * 3)()
    for e, (x, s, start) in zip(reads, ((m, a, 0), (other, b, 200), (m, a, 49))):
        e.kv, e.sequence, e.start, e.count, e.tokens = x.pool.handle, s, start, 5, tokens
    k, v = (np.zeros((15, KVH * DIM), np.float32) for _ in range(2))
    status = host.lib.safetyraise_kernel_kv_gather(host.context, reads, 3, k.ctypes.data, v.ctypes.data, 0)
    assert status == 0
    want = [x.held[s][0][[start + t for t in tokens]] for x, s, start in ((m, a, 0), (other, b, 200), (m, a, 49))]
    assert np.array_equal(k, np.concatenate(want)) and np.array_equal(v, -k)


def test_no_copies_from_nowhere(host):  # noqa: F811
    """Entries without pages or tokens copy nothing (a copy of no bytes may not name no
    address either)."""
    m = Model(host)
    a, b, c = m.new(40), m.new(20), m.new(0)
    before = host.test.test_null_copies()
    assert call(host, [(m, a, a, 0, []), (m, b, c, 0, []), ]) == 0
    m.check()
    assert call(host, [(m, c, c, 0, []), (m, b, b, 20, [])]) == 0
    m.check()
    assert host.test.test_null_copies() == before


def test_pages_that_only_targets_share(host):  # noqa: F811
    """Targets of one call that share pages with each other alone give them up together:
    they count as free pages."""
    m = Model(host, pages=20)
    parent = m.new(128)  # 8 pages
    a, b = m.fork(parent), m.fork(parent)
    m.close(parent)
    source, other = m.new(90), m.new(90)  # 6 pages each: the pool is full
    assert m.free == 0
    scattered = list(range(0, 90, 2))  # 3 pages of their own
    assert call(host, [(m, source, a, 0, scattered), (m, other, b, 0, scattered)]) == 0
    m.check()
    m.pool.destroy()


def test_pages_that_others_share_too(host):  # noqa: F811
    """... but not where another sequence, or the entry's own source, holds them."""
    m = Model(host, pages=20)
    parent = m.new(128)
    a, b = m.fork(parent), m.fork(parent)
    source = m.new(190)  # 12 pages
    assert m.free == 0
    scattered = list(range(0, 128, 2))
    assert call(host, [(m, source, a, 0, scattered), (m, source, b, 0, scattered)]) == 4
    m.check()
    assert call(host, [(m, parent, a, 0, scattered), (m, source, b, 0, scattered)]) == 4
    m.check()
    m.close(parent)
    assert call(host, [(m, a, b, 0, scattered)]) == 4  # (a keeps the pages)
    m.check()
    assert call(host, [(m, source, a, 0, scattered), (m, source, b, 0, scattered)]) == 0
    m.check()
    m.pool.destroy()


def lists_of(m):
    """Everything of a pool that a refused call may not change."""
    return m.free, {s: m.pool.len(s) for s in m.held}


@pytest.mark.parametrize("launch", ["linear_input", "kv_moves"])
def test_a_launch_that_fails_changes_nothing(host, launch):  # noqa: F811
    """Page lists, reference counts, free pages and tables are as before the call, and the
    same call can be made again."""
    rng = np.random.default_rng(5)
    failed = 0
    for turn in range(120):
        models = [Model(host, 16, int(rng.integers(60, 130))) for _ in range(3)]
        entries = []
        for m in models:
            a, b, c = (m.new(int(rng.integers(100, 300))) for _ in range(3))
            if rng.random() < 0.6:
                m.fork(int(rng.choice([a, b, c])))
            lengths = [len(m.held[s][0]) for s in (a, b)]
            kept = [sorted(rng.choice(n - 20, int(n * rng.choice([0.4, 0.95])) - 20, replace=False).tolist())
                    for n in lengths]
            entries += [(m, a, a, 20, kept[0]), (m, b, c, 20, kept[1])]
        before = [lists_of(m) for m in models]
        host.test.test_fail(launch.encode(), 0)
        status = call(host, entries)
        if host.test.test_failing():  # too few pages; or few enough tokens for the arguments
            assert status in (0, 4)
            host.test.test_fail(b"", 0)
            continue
        assert status == 5
        failed += 1
        assert [lists_of(m) for m in models] == before
        for m in models:
            m.check()
        assert call(host, entries) == 0
        for m in models:
            m.check()
            m.pool.destroy()
    assert failed > 15


def test_words_that_nothing_guards(host):  # noqa: F811
    """Where the event that says when a call's words have been read cannot be recorded, they
    are waited for: the next call may write over them."""
    m = Model(host, pages=160)
    a, b = m.new(900), m.new(500)
    kept = [t for t in range(880) if t % 7]
    entries = [(m, a, a, 20, kept), (m, b, b, 0, list(range(0, 500, 3)))]
    rows = [np.zeros((len(kept) * 2, KVH * DIM), np.float32) for _ in range(2)]
    for _ in range(6):  # (memory for all the slots' words)
        pkg.kv_gather(host, [(m.pool, a, 20, kept), (m.pool, a, 0, kept)], *rows)
    for asynchronous in (False, True):
        waits = host.test.test_waits()
        host.test.test_fail(b"event", 0)
        before = lists_of(m)
        keeps = [(x.pool, *rest) for x, *rest in entries]
        with pytest.raises(pkg.PluginError, match="hipEventRecord"):
            pkg.kv_compact(host, keeps, asynchronous=asynchronous)
        assert host.test.test_waits() > waits and lists_of(m) == before
        m.check()
    assert call(host, entries) == 0
    m.check()


def test_a_page_table_launch_that_fails(host):  # noqa: F811
    """The tokens have moved in place by then: the call reports the error, and the
    sequences are what it made them."""
    m = Model(host, pages=160)
    a, b = m.new(900), m.new(200)
    kept = [t for t in range(880) if not 30 <= t < 130]
    host.test.test_fail(b"kv_links", 0)
    rows = m.kept(a, 20, kept), m.kept(b, 7, [100, 101, 190])
    assert call(host, [(m, a, a, 20, kept), (m, b, b, 7, [100, 101, 190])]) == 5
    assert not host.test.test_failing()
    m.held[a], m.held[b] = rows
    m.check()
    m.append(a, 50)
    m.check()


def test_gather_past_a_launch(host):  # noqa: F811
    """More workgroups than a launch has are refused."""
    pool = pkg.KvCache(host, 1, 510, 16, 1, 16, 1)
    s = pool.open()
    rows = np.zeros((1, 510), np.float32)
    pool.append(s, rows, rows)
    reads = (pkg.plugin.KvRows * 1)()
    count = 1 << 25  # two tokens to a workgroup
    tokens = (C.c_uint32 * count)()
    reads[0].kv, reads[0].sequence, reads[0].count, reads[0].tokens = pool.handle, s, count, tokens
    assert host.lib.safetyraise_kernel_kv_gather(host.context, reads, 1, rows.ctypes.data, rows.ctypes.data, 0) == 3
    pool.destroy()
