"""The host rules of kv_compact (csrc/kv_plan.hpp) and of the tree calls
(csrc/tree_plan.hpp), without a GPU."""
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstring>
#include "kv_plan.hpp"
#include "tree_plan.hpp"
static int compact() {
    unsigned page, into; unsigned long long free, start, count, pages;
    while (scanf("%u %u %llu %llu %llu %llu", &page, &into, &free, &pages, &start, &count) == 6) {
        std::vector<uint32_t> tokens(count + 1), w(pages + 1);
        for (unsigned long long i = 0; i < pages; ++i) if (scanf("%u", &w[i]) != 1) return 1;
        for (unsigned long long i = 0; i < count; ++i) if (scanf("%u", &tokens[i]) != 1) return 1;
        const sr::KeepList k{start, count, tokens.data()};
        const sr::CompactPlan p = sr::compact_plan(k, page, into != 0, free, [&](uint64_t q) { return w[q] != 0; });
        printf("%llu %llu %d %zu %zu", (unsigned long long)p.first, (unsigned long long)p.fresh, (int)p.serial,
               p.take.size(), p.ranges.size());
        for (int64_t t : p.take) printf(" %lld", (long long)t);
        for (const auto &r : p.ranges) printf(" %llu %llu", (unsigned long long)r.begin, (unsigned long long)r.end);
        printf("\n");
    }
    return 0;
}
static int tree() {
    unsigned heads, kv, dim, page, n;
    while (scanf("%u %u %u %u %u", &heads, &kv, &dim, &page, &n) == 5) {
        sr::SeqMeta m[64] = {};
        for (unsigned i = 0; i < n; ++i) if (scanf("%u %u", &m[i].ctx, &m[i].rows) != 2) return 1;
        const sr::TreePlan p = sr::tree_plan(heads, kv, dim, page, 256, m, (int)n);
        printf("%d %llu", (int)p.direct, (unsigned long long)p.record_bytes);
        for (unsigned i = 0; i < n; ++i) {
            const unsigned keys = m[i].ctx + m[i].rows;
            const unsigned parts = sr::tree_parts(p, dim, keys, m[i].rows * (heads / kv));
            printf(" %u %u", parts, sr::tree_part_keys(keys, parts, dim));
        }
        printf("\n");
    }
    return 0;
}
static int valid() {
    int n;
    while (scanf("%d", &n) == 1) {
        std::vector<int32_t> p(n + 1);
        for (int i = 0; i < n; ++i) if (scanf("%d", &p[i]) != 1) return 1;
        const bool ok = sr::tree_valid(p.data(), (uint32_t)n);
        printf("%d %llu\n", (int)ok, ok && n ? (unsigned long long)sr::tree_path(p.data(), n - 1) : 0ull);
    }
    return 0;
}
int main(int, char **argv) {
    return !strcmp(argv[1], "compact") ? compact() : !strcmp(argv[1], "tree") ? tree() : valid();
}
"""


@pytest.fixture(scope="session")
def ask(tmp_path_factory):
    where = tmp_path_factory.mktemp("tree_plan")
    (where / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{ROOT / 'include'}", f"-I{ROOT / 'safetyraise-lmengine_amd' / 'csrc'}",
                    str(where / "plan.cpp"), "-o", str(where / "plan")], check=True)

    def run(what, lines):
        out = subprocess.run([str(where / "plan"), what], input="\n".join(lines) + "\n",
                             capture_output=True, text=True, check=True).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]

    return run


def compactions(seed, n):
    rng = random.Random(seed)
    for _ in range(n):
        page = rng.choice([16, 64])
        length = rng.choice([0, 1, page, 5 * page, rng.randint(1, 900)])
        start = rng.choice([0, length, rng.randint(0, length), length // page * page])
        keep = rng.choice([0.0, 0.05, 0.5, 0.95, 1.0])
        tokens = [t for t in range(length - start) if rng.random() < keep]
        if rng.random() < 0.5 and tokens:  # whole pages go
            lo = rng.randrange(len(tokens))
            tokens = tokens[:lo] + [t for t in tokens[lo:] if t >= tokens[lo] + 3 * page]
        pages = -(-length // page)
        write = [int(rng.random() < rng.choice([0.5, 1.0])) for _ in range(pages)]
        yield page, rng.randint(0, 1), rng.choice([0, 1, 5, 1000]), length, start, tokens, write


def test_compact_plans(ask):
    """Every plan, carried out, gives the kept tokens, whatever the order of its
    parallel ranges; pages of others are only read; and free pages are enough
    unless too few were there for any plan."""
    calls = list(compactions(1, 3000))
    answers = ask("compact", [
        f"{page} {into} {free} {len(write)} {start} {len(tokens)} " + " ".join(map(str, write + tokens))
        for page, into, free, length, start, tokens, write in calls])
    rng = random.Random(2)
    kinds = set()
    for (page, into, free, length, start, tokens, write), a in zip(calls, answers):
        first, fresh, serial, takes, count = a[:5]
        take, flat = a[5:5 + takes], a[5 + takes:]
        ranges = list(zip(flat[::2], flat[1::2]))
        assert len(ranges) == count
        new = start + len(tokens)
        pages = -(-new // page)
        assert first + takes == pages
        # physical pages: old page q is ("old", q)
        memory = {("old", q): list(range(q * page, min((q + 1) * page, length))) + [None] * page
                  for q in range(len(write))}
        now = [("old", q) for q in range(first)]
        for i, t in enumerate(take):
            now.append(("old", t) if t >= 0 else ("new", i))
            memory.setdefault(now[-1], [None] * (2 * page))
        assert sum(t < 0 for t in take) == fresh
        assert len(set(now)) == len(now)
        before = {p: list(x) for p, x in memory.items()}

        def source(t):
            s = t if t < start else start + tokens[t - start]
            return ("old", s // page), s % page

        order = list(ranges)
        if not serial:
            rng.shuffle(order)
        for lo, hi in order:
            step = rng.choice([1, 7, 64])
            for at in range(lo, hi, step):
                held = [memory[p][o] for p, o in (source(t) for t in range(at, min(at + step, hi)))]
                for t, x in zip(range(at, min(at + step, hi)), held):
                    memory[now[t // page]][t % page] = x
        for t in range(new):
            assert memory[now[t // page]][t % page] == (t if t < start else start + tokens[t - start])
        for q, w in enumerate(write):
            if not w or not into:
                assert memory["old", q] == before["old", q]
        if serial:
            assert into
        kinds.add((bool(serial), bool(into), fresh > 0, any(t >= 0 and t != first + i for i, t in enumerate(take))))
    assert len(kinds) >= 8


def test_tree_plans(ask):
    rng = random.Random(3)
    calls = []
    for _ in range(500):
        kv = rng.choice([1, 2, 8])
        n = rng.choice([1, 1, 2, 8, 32])
        calls.append((kv * rng.choice([1, 4, 7, 8, 12]), kv, rng.choice([64, 128, 256]), rng.choice([16, 64, 1024]),
                      [(rng.choice([0, 5, 300, 5000, rng.randint(0, 1 << 17)]), rng.randint(1, 128)) for _ in range(n)]))
    answers = ask("tree", [f"{h} {kv} {d} {p} {len(s)} " + " ".join(f"{c} {r}" for c, r in s)
                           for h, kv, d, p, s in calls])
    for (heads, kv, dim, page, seqs), (direct, record_bytes, *parts) in zip(calls, answers):
        stage = 8192 // dim
        for (context, rows), n, part in zip(seqs, parts[::2], parts[1::2]):
            assert part % stage == 0 and (n - 1) * part < context + rows <= n * part
            assert part // page + 2 <= 1024  # the partition's page ids fit in LDS
        assert bool(direct) == (max(parts[::2]) == 1)
        want = 0 if direct else sum(n * r for n, (_, r) in zip(parts[::2], seqs)) * heads * (dim + 4) * 4
        assert record_bytes == want


def test_tree_shapes(ask):
    got = ask("valid", ["3 -1 0 1", "3 -1 -1 -1", "4 -1 0 0 2", "1 0", "2 -1 1", "2 -1 -2", "1 -1"])
    assert got == [[1, 0b111], [1, 0b100], [1, 0b1101], [0, 0], [0, 0], [0, 0], [1, 1]]
