"""The operators of tree-drafted decoding, as cases for timing.

A draft model proposes a tree of tokens behind each sequence's context.  One
pass of the target model verifies every node (attention_tree_forward on the
attention layers, gdn_tree_forward on the recurrent ones), the accepted path
is committed (kv_compact, gdn_tree_commit), and kept tokens leave the cache for
another place (kv_gather).

`own` false: the operators in plain torch, over dense caches and states.
`own` true: the C entry points of this library (safetyraise_kernel_*), with
argument structs built beforehand, as the engine that loads it calls them.
"""
import ctypes as C
import importlib
import math
import random

import torch

own = False

# heads, KV heads, head_dim, rotary_dim, RoPE theta, QK-norm, gated (q and gate
# interleaved per head, norm weights with an offset of one)
SHAPES = {
    "qwen2-0.5b": (14, 2, 64, 64, 1e6, False, False),
    "qwen3-8b": (32, 8, 128, 128, 1e6, True, False),
    "qwen3-32b": (64, 8, 128, 128, 1e6, True, False),
    "qwen3.5": (16, 2, 256, 64, 1e7, True, True),
}
EPS = 1e-6
DIM = 128   # GDN key and value width
CONV = 4    # GDN conv kernel
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def attention(name, shape, seqs, context, rows, depth, page=64, scattered=False, inputs="f32",
              out="f32", mix=1):
    """`seqs` sequences of `context` (lo, hi) cached tokens, each with a tree of
    `rows` (lo, hi) drafts at most `depth` deep."""
    case = {"kind": "attention", "shape": shape, "seqs": seqs, "context_lo": context[0],
            "context_hi": context[1], "rows_lo": rows[0], "rows_hi": rows[1], "depth": depth,
            "page": page, "scattered": scattered, "inputs": inputs, "out": out, "mix": mix}
    return dict(case, name=name) if name else case


def gdn(kind, name, key_heads, value_heads, seqs, rows, depth, layers=1, inputs="f32", mix=1):
    case = {"kind": kind, "key_heads": key_heads, "value_heads": value_heads, "seqs": seqs,
            "rows_lo": rows[0], "rows_hi": rows[1], "depth": depth, "layers": layers,
            "inputs": inputs, "mix": mix}
    return dict(case, name=name) if name else case


def cache(kind, name, shape, seqs, context, kept, layers=1, page=64, scattered=False, out="bf16",
          mix=1):
    """`kept` (lo, hi): how many tokens of the compacted or gathered part stay."""
    case = {"kind": kind, "shape": shape, "seqs": seqs, "context_lo": context[0],
            "context_hi": context[1], "kept_lo": kept[0], "kept_hi": kept[1], "layers": layers,
            "page": page, "scattered": scattered, "out": out, "mix": mix}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the smallest verify: six drafts behind one short chat
        attention("tree_one", "qwen2-0.5b", 1, (300, 300), (6, 6), 3),
        # a batch of chats, each with its own tree, context 1 K to 16 K
        attention("tree_batch", "qwen3-8b", 8, (1024, 16384), (16, 32), 7, mix=2),
        # large trees behind long contexts on the hybrid model's attention
        # layers, pages scattered as in a server that has run for long
        attention("tree_hybrid", "qwen3.5", 4, (8192, 65536), (20, 64), 9, page=16,
                  scattered=True, inputs="bf16", out="bf16", mix=3),
        # a few drafts, odd lengths, many query heads to a KV head
        attention("tree_odd", "qwen3-32b", 3, (257, 3001), (1, 13), 5, inputs="bf16", mix=4),
        # one tree through one recurrent layer
        gdn("gdn_tree", "gdn_tree_one", 16, 32, 1, (12, 12), 4),
        # large trees of a batch through two recurrent layers
        gdn("gdn_tree", "gdn_tree_batch", 16, 32, 8, (24, 64), 9, layers=2, mix=2),
        # the accepted path of one sequence, one layer
        gdn("gdn_commit", "gdn_commit_one", 16, 32, 1, (12, 12), 4),
        # the accepted paths of a batch in eight recurrent layers
        gdn("gdn_commit", "gdn_commit_layers", 16, 32, 4, (24, 32), 8, layers=8, mix=2),
        # one sequence's accepted path moved into place behind its context
        cache("commit", "kv_commit_one", "qwen3-8b", 1, (1000, 1000), (4, 4)),
        # the accepted paths of a batch in every layer, into the next state of a
        # transactional engine
        cache("compact", "kv_commit_layers", "qwen3-8b", 4, (200, 700), (3, 9), layers=36, mix=2),
        # a long context thinned to the tokens that matter
        cache("compact", "kv_evict", "qwen3-8b", 2, (20001, 32768), (5000, 8192), scattered=True,
              mix=3),
        # chosen tokens of long contexts copied out for another place, in f32
        cache("gather", "kv_gather", "qwen3.5", 3, (9000, 40000), (4000, 16001), page=16,
              scattered=True, out="f32", mix=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "gdn_tree", "gdn_tree", "gdn_commit",
                       "commit", "compact", "gather"])
    mix = rng.randrange(1, 1 << 16)
    inputs = rng.choice(["f32", "bf16"])
    page, scattered = rng.choice([16, 64]), rng.random() < 0.5
    if kind == "attention":
        shape = rng.choice(list(SHAPES))
        heads, kvh, dim = SHAPES[shape][:3]
        seqs, rows = _log(rng, 1, 12), _log(rng, 2, 64)
        most = min(65536, 1.2e8 / (kvh * dim * seqs), 6e9 / (heads * dim * rows * seqs) * 4)
        hi = max(280, min(_log(rng, 280, 65536), int(most)))
        return attention(None, shape, seqs, (max(260, hi // rng.randint(1, 12)), hi),
                         (max(1, rows // rng.randint(1, 4)), rows), rng.randint(1, 10), page=page,
                         scattered=scattered, inputs=inputs, out=rng.choice(["f32", "bf16"]),
                         mix=mix)
    if kind.startswith("gdn"):
        key_heads = rng.choice([4, 8, 16])
        value_heads = key_heads * rng.choice([1, 2, 2, 4]) if key_heads < 16 else rng.choice([16, 32])
        rows = _log(rng, 2, 64)
        seqs = _log(rng, 1, 8)
        layers = rng.randint(1, 2) if kind == "gdn_tree" else rng.randint(1, 8)
        if kind == "gdn_commit":
            seqs, rows = min(seqs, 4), min(rows, 32)
        return gdn(kind, None, key_heads, value_heads, seqs, (max(1, rows // rng.randint(1, 4)), rows),
                   rng.randint(1, 10), layers=layers, inputs=inputs, mix=mix)
    shape = rng.choice(list(SHAPES))
    kvh, dim = SHAPES[shape][1:3]
    out = rng.choice(["f32", "bf16"])
    if kind == "commit":
        return cache(kind, None, shape, rng.randint(1, 3), (260, _log(rng, 280, 4096)),
                     (1, rng.randint(2, 12)), page=page, scattered=scattered, out=out, mix=mix)
    if kind == "compact" and rng.random() < 0.5:
        hi = _log(rng, 64, 700)
        return cache(kind, None, shape, rng.randint(1, 4), (max(32, hi // 3), hi),
                     (1, rng.randint(2, 16)), layers=rng.randint(2, 36), page=page,
                     scattered=scattered, out=out, mix=mix)
    seqs = rng.randint(1, 3)
    hi = min(_log(rng, 300, 40000), int(6e7 / (kvh * dim * seqs)))
    kept = max(2, int(hi * rng.uniform(0.05, 0.4)))
    return cache(kind, None, shape, seqs, (max(150, hi // 2), hi), (kept // 2, kept), page=page,
                 scattered=scattered, out=out, mix=mix)


# ------------------------------------------------------- what the cases share

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _between(case, what):
    """One whole number per sequence in [what_lo, what_hi], fixed by the case."""
    r = random.Random("%s %d" % (what, case["mix"]))
    lo, hi = case[what + "_lo"], case[what + "_hi"]
    n = [r.randint(lo, hi) for _ in range(case["seqs"])]
    n[-1] = hi
    return n


def _trees(case):
    """Per sequence the parents of its drafts: -1 behind the context."""
    r = random.Random("tree %d" % case["mix"])
    trees = []
    for rows in _between(case, "rows"):
        parents, depths = [], []
        for i in range(rows):
            p = -1 if i == 0 or r.random() < 0.15 else r.randrange(max(0, i - 12), i)
            if p >= 0 and depths[p] + 1 >= case["depth"]:
                p = parents[p]
            parents.append(p)
            depths.append(0 if p < 0 else depths[p] + 1)
        trees.append(parents)
    return trees


def _path(parents, row):
    """The rows from the root down to `row`."""
    path = []
    while row >= 0:
        path.append(row)
        row = parents[row]
    return path[::-1]


def _accepted(parents):
    """A deepest draft: the end of the path that is committed."""
    return max(range(len(parents)), key=lambda i: (len(_path(parents, i)), -i))


def _dev(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device="cuda")


class State:
    """Inputs, handles and prebuilt calls of one prepared case."""

    def __init__(self, case):
        self.case = case
        self.owned = []
        self.keep = []
        self.calls = []

    def __del__(self):
        for o in self.owned:
            o.destroy()


class Held(list):
    """Outputs in a pool's own memory, which lives as long as they do."""

    def __init__(self, outputs, state):
        super().__init__(outputs)
        self.state = state


_backend = None


def _engine():
    """The package and the process's context, made once as an engine does."""
    global _backend
    pkg = importlib.import_module("safetyraise-lmengine_amd")
    if _backend is None:
        _backend = pkg.NativeBackend.load()
    return pkg, pkg.plugin, _backend


def _u32(values):
    return (C.c_uint32 * len(values))(*values)


def _i32(values):
    return (C.c_int32 * len(values))(*values)


def _rms(x, weight):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


# ------------------------------------------------------------------ attention

def _attention_inputs(case, seed):
    heads, kvh, dim, rot, theta, norm, gated = SHAPES[case["shape"]]
    g = _gen(seed)
    dtype = TYPES[case["inputs"]]
    contexts, trees = _between(case, "context"), _trees(case)
    ck, cv = (_randn(g, (case["seqs"], max(contexts), kvh, dim), torch.bfloat16) for _ in range(2))
    total = sum(len(t) for t in trees)
    q = _randn(g, (total, heads * dim * (2 if gated else 1)), dtype)
    k, v = (_randn(g, (total, kvh * dim), dtype) for _ in range(2))
    gains = [(0.0 if gated else 1.0) + 0.02 * _randn(g, (dim,)) for _ in range(2)]
    positions = [n + len(_path(t, i)) - 1 for n, t in zip(contexts, trees) for i in range(len(t))]
    pos = _dev(positions, torch.int32).view(-1, 1).repeat(1, 3).contiguous()
    return contexts, trees, ck, cv, q, k, v, gains, pos


def _pool_of(pkg, backend, case, layers, lengths, room):
    """One KV pool per layer with a sequence for each length, and `room` more
    sequences of that size."""
    kvh, dim = SHAPES[case["shape"]][1:3]
    page, most = case["page"], max(lengths)
    pages = (1 + room) * case["seqs"] * (most // page + 2) + 8
    return [pkg.KvCache(backend, kvh, dim, page, pages, most + 1, (1 + room) * case["seqs"],
                        page_order_seed=1 + (case["mix"] + i) % 65535 if case["scattered"] else 0)
            for i in range(layers)]


def _prepare_attention(case, seed):
    heads, kvh, dim, rot, theta, norm, gated = SHAPES[case["shape"]]
    contexts, trees, ck, cv, q, k, v, gains, pos = _attention_inputs(case, seed)
    s = State(case)
    s.q, s.k, s.v, s.gains, s.pos = q, k, v, gains, pos
    if not own:
        rows, most = max(len(t) for t in trees), max(n + len(t) for n, t in zip(contexts, trees))
        s.keys, s.values = (torch.cat([c, c.new_zeros((c.shape[0], most - c.shape[1]) + c.shape[2:])], 1)
                            for c in (ck, cv))
        s.seq = _dev([i for i, t in enumerate(trees) for _ in t])
        s.row = _dev([r for t in trees for r in range(len(t))])
        s.slot = _dev([n + r for n, t in zip(contexts, trees) for r in range(len(t))])
        see = torch.zeros((case["seqs"], rows, most), dtype=torch.bool)
        for i, (n, t) in enumerate(zip(contexts, trees)):
            see[i, :, :n] = True
            for r in range(len(t)):
                see[i, r, [n + j for j in _path(t, r)]] = True
        s.visible = see.cuda()
        return s
    pkg, P, backend = _engine()
    pool, = _pool_of(pkg, backend, case, 1, [n + len(t) for n, t in zip(contexts, trees)], 0)
    s.owned.append(pool)
    ids = [pool.open() for _ in contexts]
    for i, n in enumerate(contexts):
        pool.append(ids[i], ck[i, :n].reshape(n, -1), cv[i, :n].reshape(n, -1))
    s.out = torch.empty((q.shape[0], heads * dim), device="cuda", dtype=TYPES[case["out"]])
    a = P.AttentionTreeArgs()
    a.struct_size = C.sizeof(a)
    b = a.attention
    b.struct_size = C.sizeof(b)
    b.flags = P.DEVICE_POINTERS | P.ASYNC | P.MROPE_INTERLEAVED
    b.flags |= P.INPUT_BF16 if case["inputs"] == "bf16" else 0
    b.flags |= P.OUTPUT_BF16 if case["out"] == "bf16" else 0
    b.flags |= P.QK_NORM if norm else 0
    b.flags |= P.GATED | P.NORM_OFFSET if gated else 0
    b.heads, b.kv_heads, b.head_dim, b.rotary_dim = heads, kvh, dim, rot
    b.eps, b.rope_theta, b.num_seqs = EPS, theta, len(ids)
    s.keep += [_u32(ids), _u32([len(t) for t in trees]), _i32([p for t in trees for p in t]), a]
    b.seq_ids, b.seq_rows, a.parents = s.keep[:3]
    b.q, b.k, b.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if norm:
        b.q_norm, b.k_norm = gains[0].data_ptr(), gains[1].data_ptr()
    b.positions, b.out, b.kv = pos.data_ptr(), s.out.data_ptr(), pool.handle
    lib, ctx = backend.lib, backend.context
    s.calls.append((lib.safetyraise_kernel_attention_tree_forward, (ctx, C.byref(a))))
    # the drafts are taken back, so that the next pass starts from the same contexts
    s.calls += [(lib.safetyraise_kernel_kv_truncate, (ctx, pool.handle, i, n))
                for i, n in zip(ids, contexts)]
    return s


def _angles(pos, theta, rot):
    """The path's own angle: an f32 position over an f32 power of theta."""
    power = torch.tensor([math.pow(theta, 2 * i / rot) for i in range(rot // 2)],
                         dtype=torch.float32, device=pos.device)
    return (pos[:, :1].float() / power).double()


def _rope(x, angle, rot):
    c, s = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
    left, right = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([left * c - right * s, right * c + left * s, x[..., rot:]], -1)


def _plain_attention(s):
    heads, kvh, dim, rot, theta, norm, gated = SHAPES[s.case["shape"]]
    total, group = s.q.shape[0], heads // kvh
    q, k = s.q.float().view(total, heads, -1), s.k.float().view(total, kvh, dim)
    if gated:
        q, gate = q[..., :dim], q[..., dim:]
    if norm:
        q, k = (_rms(x, w + (1.0 if gated else 0.0)) for x, w in zip((q, k), s.gains))
    angle = _angles(s.pos, theta, rot)
    q, k = _rope(q, angle, rot), _rope(k, angle, rot)
    keys, values = s.keys.float(), s.values.float()
    keys[s.seq, s.slot] = k.to(torch.bfloat16).float()
    values[s.seq, s.slot] = s.v.to(torch.bfloat16).float().view(total, kvh, dim)
    n, rows, most = s.visible.shape
    batch = q.new_zeros((n, rows, kvh, group, dim))
    batch[s.seq, s.row] = q.view(total, kvh, group, dim)
    batch = batch.permute(0, 2, 3, 1, 4).reshape(n, kvh, group * rows, dim)
    score = (batch @ keys.permute(0, 2, 3, 1).contiguous()) / math.sqrt(dim)
    score = score.view(n, kvh, group, rows, most).masked_fill_(~s.visible[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True)).view(n, kvh, group * rows, most)
    out = (p @ values.permute(0, 2, 1, 3).contiguous()) / p.sum(-1, keepdim=True)
    out = out.view(n, kvh, group, rows, dim).permute(0, 3, 1, 2, 4).reshape(n, rows, heads, dim)
    out = out[s.seq, s.row]
    if gated:
        out = out * torch.sigmoid(gate)
    return out.reshape(total, heads * dim).to(TYPES[s.case["out"]])


def _exact_attention(case, seed):
    heads, kvh, dim, rot, theta, norm, gated = SHAPES[case["shape"]]
    group = heads // kvh
    contexts, trees, ck, cv, q, k, v, gains, pos = _attention_inputs(case, seed)
    total = q.shape[0]
    q, k, v = (x.double() for x in (q, k, v))
    q, k = q.view(total, heads, -1), k.view(total, kvh, dim)
    gate = q[..., dim:] if gated else None
    q = q[..., :dim]
    if norm:
        offset = 1.0 if gated else 0.0
        q, k = _rms(q, gains[0].double() + offset), _rms(k, gains[1].double() + offset)
    angle = _angles(pos, theta, rot)
    q, k = _rope(q, angle, rot), _rope(k, angle, rot)
    # the cache holds bf16
    k, v = k.to(torch.bfloat16).double(), v.to(torch.bfloat16).double().view(total, kvh, dim)
    out = torch.empty((total, heads, dim), dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, tree) in enumerate(zip(contexts, trees)):
        rows = slice(at, at + len(tree))
        at += len(tree)
        hidden = torch.ones((len(tree), n + len(tree)), dtype=torch.bool)
        hidden[:, :n] = False
        for r in range(len(tree)):
            hidden[r, [n + j for j in _path(tree, r)]] = False
        hidden = hidden.cuda()
        for h in range(kvh):
            keys = torch.cat([ck[i, :n, h].double(), k[rows, h]])
            values = torch.cat([cv[i, :n, h].double(), v[rows, h]])
            for j in range(h * group, (h + 1) * group):
                score = q[rows, j] @ keys.T / math.sqrt(dim)
                score = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[rows, j] = score @ values
    if gated:
        out *= torch.sigmoid(gate)
    return out.view(total, heads * dim)


def _work_attention(case):
    heads, kvh, dim, rot, theta, norm, gated = SHAPES[case["shape"]]
    size, wide = (2 if case[t] == "bf16" else 4 for t in ("inputs", "out"))
    moved = flops = 0
    for n, tree in zip(_between(case, "context"), _trees(case)):
        rows = len(tree)
        moved += (n + rows) * kvh * dim * 4
        moved += rows * ((heads * (2 if gated else 1) + 2 * kvh) * dim * size + heads * dim * wide + 12)
        flops += 4 * dim * heads * (n * rows + sum(len(_path(tree, r)) for r in range(rows)))
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------ GDN

def _gdn_width(case):
    hk, hv = case["key_heads"], case["value_heads"]
    return 2 * hk * DIM + hv * DIM, hv * DIM, hv


def _gdn_inputs(case, seed):
    """Per layer: weights, the states and histories before the tree, its rows.
    A decay rate per head of 1 to 16 and a step of 0.001 to 0.1, as such layers
    are initialised; conv taps of unit gain, norm weights about one."""
    channels, width, hv = _gdn_width(case)
    g = _gen(seed)
    total = sum(_between(case, "rows"))
    layers = []
    for _ in range(case["layers"]):
        a_log = torch.log(1 + 15 * torch.rand(hv, generator=g, device="cuda"))
        step = torch.exp(math.log(1e-3) + math.log(100) * torch.rand(hv, generator=g, device="cuda"))
        weights = (a_log, torch.log(torch.expm1(step)), _randn(g, (channels, CONV)) / 2,
                   1 + 0.02 * _randn(g, (DIM,)))
        state = 0.1 * _randn(g, (case["seqs"], hv, DIM, DIM))
        history = _randn(g, (case["seqs"], channels, CONV - 1))
        rows = [_randn(g, (total, n), TYPES[case["inputs"]]) for n in (channels, width, hv, hv)]
        layers.append((weights, state, history, rows))
    return layers


def _gdn_plan(case):
    """The trees as indices: where each row's conv taps and parent state are
    (histories and states of the sequences first, then the rows), and the
    rows of each level."""
    trees, taps, parent, levels, at = _trees(case), [], [], [], 0
    n = case["seqs"]
    for i, tree in enumerate(trees):
        for r in range(len(tree)):
            path = _path(tree, r)
            line = [(CONV - 1) * i + j for j in range(CONV - 1)]
            line += [(CONV - 1) * n + at + j for j in path]
            taps.append(line[-CONV:])
            parent.append(i if tree[r] < 0 else n + at + tree[r])
            levels += [[] for _ in range(len(path) - len(levels))]
            levels[len(path) - 1].append(at + r)
        at += len(tree)
    return _dev(taps), _dev(parent), [_dev(rows) for rows in levels]


def _plain_records(case, plan, weights, state, history, rows):
    """Outputs and, per row, log decay, correction and key."""
    a_log, dt_bias, taps, norm = weights
    where, parent, levels = plan
    qkv, z, a, b = (x.float() for x in rows)
    n, total, hk, hv = case["seqs"], qkv.shape[0], case["key_heads"], case["value_heads"]
    line = torch.cat([history.transpose(1, 2).reshape(n * (CONV - 1), -1), qkv])
    conv = (line[where] * taps.T).sum(1)
    conv = conv * torch.sigmoid(conv)
    q, k = (x.reshape(total, hk, DIM) for x in conv[:, :2 * hk * DIM].split(hk * DIM, 1))
    v = conv[:, 2 * hk * DIM:].reshape(total, hv, DIM)
    q, k = ((x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6)).repeat_interleave(hv // hk, 1)
            for x in (q, k))
    x = a + dt_bias
    log_alpha = -torch.exp(a_log) * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    beta = torch.sigmoid(b)[..., None]
    states = torch.cat([state, state.new_empty((total,) + state.shape[1:])])
    delta, out = torch.empty_like(v), torch.empty_like(v)
    for level in levels:
        s = states[parent[level]] * torch.exp(log_alpha[level])[..., None, None]
        d = beta[level] * (v[level] - (s @ k[level][..., None])[..., 0])
        s = s + d[..., None] * k[level][:, :, None, :]
        states[n + level] = s
        delta[level] = d
        out[level] = (s @ q[level][..., None])[..., 0] / math.sqrt(DIM)
    z = z.view(total, hv, DIM)
    out = (_rms(out, norm) * z * torch.sigmoid(z)).reshape(total, hv * DIM)
    return out, log_alpha, delta, k


def _prepare_gdn(case, seed):
    s = State(case)
    s.layers = _gdn_inputs(case, seed)
    trees, commit = _trees(case), case["kind"] == "gdn_commit"
    first = [0]
    for t in trees:
        first.append(first[-1] + len(t))
    if not own:
        s.plan = _gdn_plan(case)
        if commit:
            # the forward's records, which the commit reads, and the paths, padded
            s.records = [_plain_records(case, s.plan, *layer)[1:] for layer in s.layers]
            paths = [[first[i] + r for r in _path(t, _accepted(t))] for i, t in enumerate(trees)]
            most = max(len(p) for p in paths)
            s.path = _dev([p + [p[-1]] * (most - len(p)) for p in paths])
            s.on_path = _dev([[1.0] * len(p) + [0.0] * (most - len(p)) for p in paths], torch.float32)
            taps = [[(CONV - 1) * i + j for j in range(CONV - 1)] +
                    [(CONV - 1) * case["seqs"] + r for r in p] for i, p in enumerate(paths)]
            s.taps = _dev([t[-(CONV - 1):] for t in taps])
        return s
    pkg, P, backend = _engine()
    lib, ctx = backend.lib, backend.context
    total, width = first[-1], _gdn_width(case)[1]
    s.out = torch.empty((case["layers"], total, width), device="cuda")
    commits = (P.GdnCommit * (case["layers"] * case["seqs"]))()
    for n, (weights, state, history, rows) in enumerate(s.layers):
        pool = pkg.GdnState(backend, case["key_heads"], case["value_heads"], DIM, DIM, CONV,
                            case["seqs"], keep_rows=64)
        s.owned.append(pool)
        ids = [pool.open() for _ in trees]
        for i in ids:
            pool.write(i, state[i].cpu().numpy(), history[i].cpu().numpy())
        a = P.GdnTreeArgs()
        a.struct_size = C.sizeof(a)
        b = a.gdn
        b.struct_size = C.sizeof(b)
        b.flags = P.DEVICE_POINTERS | P.ASYNC
        b.flags |= P.INPUT_BF16 if case["inputs"] == "bf16" else 0
        b.eps, b.num_seqs = EPS, len(ids)
        keep = [_u32(ids), _u32([len(t) for t in trees]), _i32([p for t in trees for p in t]), a]
        b.seq_ids, b.seq_rows, a.parents = keep[:3]
        s.keep += keep
        b.qkv, b.z, b.a, b.b = (t.data_ptr() for t in rows)
        b.a_log, b.dt_bias, b.conv_weight, b.norm = (t.data_ptr() for t in weights)
        b.out, b.state = s.out[n].data_ptr(), pool.handle
        forward = (lib.safetyraise_kernel_gdn_tree_forward, (ctx, C.byref(a)))
        if not commit:
            s.calls.append(forward)
            continue
        backend.check(forward[0](*forward[1]), "gdn_tree_forward")
        for i, t in zip(ids, trees):
            c = commits[n * case["seqs"] + i]
            c.state, c.sequence, c.row = pool.handle, i, _accepted(t)
    if commit:
        s.keep.append(commits)
        call = (lib.safetyraise_kernel_gdn_tree_commit, (ctx, commits, len(commits), P.ASYNC))
        s.calls.append(call)
        # the committed state and history where the pools hold them
        backend.check(call[0](*call[1]), "gdn_tree_commit")
        s.out = [pool.view(i) for pool in s.owned for i in range(case["seqs"])]
    backend.synchronize()
    return s


def _plain_gdn(s):
    return torch.stack([_plain_records(s.case, s.plan, *layer)[0] for layer in s.layers])


def _plain_commit(s):
    case, out = s.case, []
    for (_, state, history, rows), (log_alpha, delta, key) in zip(s.layers, s.records):
        on = s.on_path[..., None]
        decay = torch.cumsum(log_alpha[s.path].double() * on, 1)
        last = decay[:, -1:]
        weight = (torch.exp(last - decay).float() * on)[..., None]
        new = state * torch.exp(last[:, 0]).float()[..., None, None]
        new = new + (weight * delta[s.path]).permute(0, 2, 3, 1) @ key[s.path].permute(0, 2, 1, 3)
        line = torch.cat([history.transpose(1, 2).reshape(-1, history.shape[1]), rows[0].float()])
        out += list(zip(new, line[s.taps].transpose(1, 2).contiguous()))
    return out


def _exact_gdn(case, seed):
    trees, outs = _trees(case), []
    hk, hv = case["key_heads"], case["value_heads"]
    for weights, state, history, rows in _gdn_inputs(case, seed):
        a_log, dt_bias, taps, norm = (t.double() for t in weights)
        qkv, z, a, b = (t.double() for t in rows)
        outs.append([])
        at = 0
        for i, tree in enumerate(trees):
            after = {-1: (state[i].double(), history[i].double())}
            for r in range(len(tree)):
                s, line = after[tree[r]]
                line = torch.cat([line, qkv[at + r][:, None]], 1)
                x = (line * taps).sum(1)
                x = x / (1 + torch.exp(-x))
                q, k, v = x.split([hk * DIM, hk * DIM, hv * DIM])
                q, k = (y.view(hk, DIM) / (y.view(hk, DIM).square().sum(1, keepdim=True) + 1e-6).sqrt()
                        for y in (q, k))
                q, k = q.repeat_interleave(hv // hk, 0), k.repeat_interleave(hv // hk, 0)
                step = torch.nn.functional.softplus(a[at + r] + dt_bias, threshold=1e9)
                s = s * torch.exp(-a_log.exp() * step)[:, None, None]
                miss = v.view(hv, DIM) - torch.einsum("hvk,hk->hv", s, k)
                s = s + torch.einsum("hv,hk->hvk", torch.sigmoid(b[at + r])[:, None] * miss, k)
                o = torch.einsum("hvk,hk->hv", s, q) / math.sqrt(DIM)
                o = _rms(o, norm).reshape(-1)
                outs[-1].append(o * z[at + r] / (1 + torch.exp(-z[at + r])))
                after[r] = (s, line[:, 1:])
            at += len(tree)
    return torch.stack([torch.stack(rows) for rows in outs])


def _exact_commit(case, seed):
    trees, out = _trees(case), []
    hk, hv = case["key_heads"], case["value_heads"]
    for weights, state, history, rows in _gdn_inputs(case, seed):
        a_log, dt_bias, taps, _ = (t.double() for t in weights)
        qkv, _, a, b = (t.double() for t in rows)
        at = 0
        for i, tree in enumerate(trees):
            s, line = state[i].double(), history[i].double()
            for r in _path(tree, _accepted(tree)):
                line = torch.cat([line[:, 1 - CONV:], qkv[at + r][:, None]], 1)
                x = (line * taps).sum(1)
                x = x / (1 + torch.exp(-x))
                _, k, v = x.split([hk * DIM, hk * DIM, hv * DIM])
                k = k.view(hk, DIM) / (k.view(hk, DIM).square().sum(1, keepdim=True) + 1e-6).sqrt()
                k = k.repeat_interleave(hv // hk, 0)
                step = torch.nn.functional.softplus(a[at + r] + dt_bias, threshold=1e9)
                s = s * torch.exp(-a_log.exp() * step)[:, None, None]
                miss = v.view(hv, DIM) - torch.einsum("hvk,hk->hv", s, k)
                s = s + torch.einsum("hv,hk->hvk", torch.sigmoid(b[at + r])[:, None] * miss, k)
            out.append((s, line[:, 1 - CONV:].contiguous()))
            at += len(tree)
    return out


def _work_gdn(case):
    channels, width, hv = _gdn_width(case)
    size = 2 if case["inputs"] == "bf16" else 4
    state = hv * DIM * DIM * 4 + channels * (CONV - 1) * 4
    trees, layers = _trees(case), case["layers"]
    rows = sum(len(t) for t in trees)
    if case["kind"] == "gdn_commit":
        path = sum(len(_path(t, _accepted(t))) for t in trees)
        moved = case["seqs"] * 2 * state + path * (width + case["key_heads"] * DIM + hv) * 4
        return {"bytes": layers * moved, "flops": layers * path * hv * 3 * DIM * DIM}
    moved = case["seqs"] * state + channels * CONV * 4
    moved += rows * ((channels + width + 2 * hv) * size + width * 4)
    pairs = sum(len(_path(t, r)) for t in trees for r in range(len(t)))
    return {"bytes": layers * moved, "flops": layers * hv * (rows * 4 + pairs * 8 / DIM) * DIM * DIM}


# ---------------------------------------------------------------------- cache

def _kept(case):
    """Per sequence: its length, where the compacted part starts, and the tokens
    that stay, counted from there."""
    r = random.Random("kept %d" % case["mix"])
    plans = []
    for n, kept in zip(_between(case, "context"), _between(case, "kept")):
        if case["kind"] == "gather" or case["layers"] == 1 and case["kind"] == "compact":
            # the first tokens, the latest, and scattered ones between
            edge = max(1, kept // 8)
            few = list(range(min(4, edge))) + list(range(n - edge, n))
            tokens = sorted(set(few + r.sample(range(n), max(0, kept - len(few)))))
            plans.append((n, 0, tokens))
        else:
            # the accepted path among the drafts behind the context
            drafts = 3 * kept
            plans.append((n + drafts, n, sorted(r.sample(range(drafts), kept))))
    return plans


def _cache_inputs(case, seed):
    kvh, dim = SHAPES[case["shape"]][1:3]
    g = _gen(seed)
    shape = (case["layers"], case["seqs"], max(n for n, _, _ in _kept(case)), kvh, dim)
    return [_randn(g, shape, torch.bfloat16) for _ in range(2)]


def _prepare_cache(case, seed):
    kvh, dim = SHAPES[case["shape"]][1:3]
    plans, kind, seqs = _kept(case), case["kind"], case["seqs"]
    s = State(case)
    s.cache = _cache_inputs(case, seed)
    kept = sum(len(t) for _, _, t in plans)
    if not own:
        s.seq = _dev([i for i, (_, _, t) in enumerate(plans) for _ in t])
        s.src = _dev([at + j for _, at, t in plans for j in t])
        s.dst = _dev([at + j for _, at, t in plans for j in range(len(t))])
        if kind == "compact":
            s.target = [torch.empty_like(c) for c in s.cache]
        if kind == "commit":
            s.draft_seq = _dev([i for i, (n, at, _) in enumerate(plans) for _ in range(at, n)])
            s.draft_slot = _dev([j for n, at, _ in plans for j in range(at, n)])
            s.drafts = [c[:, s.draft_seq, s.draft_slot] for c in s.cache]
        return s
    pkg, P, backend = _engine()
    lib, ctx = backend.lib, backend.context
    pools = _pool_of(pkg, backend, case, case["layers"], [n for n, _, _ in plans],
                     1 if kind == "compact" else 0)
    s.owned += pools
    s.out = [torch.empty((case["layers"], kept, kvh, dim), device="cuda", dtype=TYPES[case["out"]])
             for _ in range(2)]
    keeps = (P.KvKeep * (case["layers"] * seqs))()
    reads = (P.KvRows * (case["layers"] * seqs))()
    tokens = [_u32(t) for _, _, t in plans]
    s.keep += [keeps, reads, tokens]
    for layer, pool in enumerate(pools):
        ids = [pool.open() for _ in plans]
        into = [pool.open() for _ in plans] if kind == "compact" else ids
        for i, (n, at, t) in enumerate(plans):
            k, v = (c[layer, i, :n].reshape(n, -1) for c in s.cache)
            pool.append(ids[i], k, v)
            x, y = keeps[layer * seqs + i], reads[layer * seqs + i]
            x.kv, x.source, x.target, x.start = pool.handle, ids[i], into[i], at
            x.count, x.tokens = len(t), tokens[i]
            y.kv, y.sequence, y.start, y.count = pool.handle, into[i], at, len(t)
            if kind == "gather":
                y.tokens = tokens[i]
            if kind == "commit":
                # the drafts again, as the next verify writes them
                s.calls.append((lib.safetyraise_kernel_kv_truncate, (ctx, pool.handle, ids[i], at)))
                s.calls.append((lib.safetyraise_kernel_kv_append,
                                (ctx, pool.handle, ids[i], k[at:].data_ptr(), v[at:].data_ptr(),
                                 n - at, P.DEVICE_POINTERS | P.ASYNC | P.INPUT_BF16)))
    if kind != "gather":
        s.calls.append((lib.safetyraise_kernel_kv_compact, (ctx, keeps, len(keeps), P.ASYNC)))
    flags = P.DEVICE_POINTERS | P.ASYNC | (P.OUTPUT_BF16 if case["out"] == "bf16" else 0)
    s.calls.append((lib.safetyraise_kernel_kv_gather,
                    (ctx, reads, len(reads), s.out[0].data_ptr(), s.out[1].data_ptr(), flags)))
    return s


def _plain_cache(s):
    if s.case["kind"] == "commit":
        # the drafts, as the verify writes them, then the kept ones in front
        for t, x in zip(s.cache, s.drafts):
            t[:, s.draft_seq, s.draft_slot] = x
    out = [c[:, s.seq, s.src] for c in s.cache]
    if s.case["kind"] != "gather":
        target = s.target if s.case["kind"] == "compact" else s.cache
        for t, x in zip(target, out):
            t[:, s.seq, s.dst] = x
        out = [t[:, s.seq, s.dst] for t in target]
    return [x.to(TYPES[s.case["out"]]) for x in out]


def _exact_cache(case, seed):
    return [torch.cat([torch.stack([c[layer, i, at + torch.tensor(t, device="cuda")].double()
                                    for layer in range(case["layers"])])
                       for i, (_, at, t) in enumerate(_kept(case))], 1)
            for c in _cache_inputs(case, seed)]


def _work_cache(case):
    kvh, dim = SHAPES[case["shape"]][1:3]
    plans = _kept(case)
    kept = case["layers"] * sum(len(t) for _, _, t in plans)
    row = 2 * kvh * dim  # values of a token
    moved = kept * row * (2 + (2 if case["out"] == "bf16" else 4))
    if case["kind"] != "gather":
        moved += kept * row * 4
    if case["kind"] == "commit":
        moved += sum(n - at for n, at, _ in plans) * row * 4
    return {"bytes": moved, "flops": 0}


# ----------------------------------------------------------------- the module

def prepare(case, seed):
    if case["kind"] == "attention":
        s = _prepare_attention(case, seed)
    elif case["kind"].startswith("gdn"):
        s = _prepare_gdn(case, seed)
    else:
        s = _prepare_cache(case, seed)
    torch.cuda.synchronize()
    return s


def run(state):
    if not own:
        kind = state.case["kind"]
        if kind == "attention":
            return _plain_attention(state)
        if kind.startswith("gdn"):
            return _plain_gdn(state) if kind == "gdn_tree" else _plain_commit(state)
        return _plain_cache(state)
    for call, arguments in state.calls:
        status = call(*arguments)
        if status:
            _backend.check(status, call.__name__)
    return Held(state.out, state) if state.case["kind"] == "gdn_commit" else state.out


def work(case):
    if case["kind"] == "attention":
        return _work_attention(case)
    return _work_gdn(case) if case["kind"].startswith("gdn") else _work_cache(case)


def exact(case, seed):
    if case["kind"] == "attention":
        return _exact_attention(case, seed)
    if case["kind"].startswith("gdn"):
        return _exact_gdn(case, seed) if case["kind"] == "gdn_tree" else _exact_commit(case, seed)
    return _exact_cache(case, seed)
