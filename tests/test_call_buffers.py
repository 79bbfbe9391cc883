"""What the Python entry points check of their buffers before the library is called,
without a GPU: a stub in the library's place that must not be reached."""
import importlib
import types

import numpy as np
import pytest
import torch

pkg = importlib.import_module("safetyraise-lmengine_amd")
HEADS, KVH, DIM, ROWS = 4, 2, 16, 3


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


class Device(torch.Tensor):
    """A host tensor that says it is on a GPU."""
    is_cuda = True


@pytest.fixture
def backend():
    return types.SimpleNamespace(lib=Library(), context=1, stream=None, check=lambda status, what: None)


def floats(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def attention_args():
    return dict(q=floats(ROWS, HEADS * DIM), k=floats(ROWS, KVH * DIM), v=floats(ROWS, KVH * DIM),
                positions=torch.zeros((ROWS, 3), dtype=torch.int32), out=floats(ROWS, HEADS * DIM),
                q_norm=floats(DIM), k_norm=floats(DIM))


def run_attention(backend, tree=True, **change):
    kv = types.SimpleNamespace(handle=1)
    args = dict(attention_args(), **change)
    common = dict(args, heads=HEADS, kv_heads=KVH, head_dim=DIM, rotary_dim=DIM, rope_theta=1e4)
    if tree:
        pkg.attention_tree_forward(backend, kv, [0], [ROWS], [-1, 0, 0], **common)
    else:
        pkg.attention_forward(backend, kv, [0], [ROWS], **common)


def bf16(x):
    return x.bfloat16()


def short(x):
    return x.reshape(-1)[:-1]


def on_device(x):
    return x.as_subclass(Device)


@pytest.mark.parametrize("name,how,error", [
    ("out", short, ValueError), ("out", torch.Tensor.half, TypeError), ("out", torch.Tensor.double, TypeError),
    ("q", short, ValueError), ("q", torch.Tensor.half, TypeError), ("k", bf16, TypeError), ("v", bf16, TypeError),
    ("k", short, ValueError), ("v", short, ValueError), ("positions", torch.Tensor.long, TypeError),
    ("positions", short, ValueError), ("q_norm", bf16, TypeError), ("k_norm", short, ValueError),
    ("out", on_device, ValueError), ("v", on_device, ValueError),
])
def test_attention_tree_refuses(backend, name, how, error):
    with pytest.raises(error, match=name):
        run_attention(backend, **{name: how(attention_args()[name])})
    assert not backend.lib.calls


def test_attention_tree_takes(backend):
    run_attention(backend)
    run_attention(backend, out=bf16(attention_args()["out"]))
    run_attention(backend, **{n: bf16(attention_args()[n]) for n in "qkv"})
    run_attention(backend, q_norm=None, k_norm=None)
    run_attention(backend, out=floats(ROWS + 1, HEADS * DIM))
    run_attention(backend, **{n: x.numpy() for n, x in attention_args().items()})
    assert len(backend.lib.calls) == 6
    with pytest.raises(ValueError, match="q has"):
        backend.lib.calls.clear()
        kv = types.SimpleNamespace(handle=1)
        pkg.attention_tree_forward(backend, kv, [0], [ROWS], [-1, 0, 0], **attention_args(), gated=True,
                                   heads=HEADS, kv_heads=KVH, head_dim=DIM, rotary_dim=DIM, rope_theta=1e4)


def test_results_that_are_always_float32(backend):
    """attention_forward and gdn_forward write float32, whatever out is."""
    with pytest.raises(TypeError, match="out is bfloat16"):
        run_attention(backend, tree=False, out=bf16(attention_args()["out"]))
    with pytest.raises(TypeError, match="out is bfloat16"):
        run_gdn(backend, pkg.gdn_forward, out=bf16(gdn_args()["out"]))
    assert not backend.lib.calls
    run_attention(backend, tree=False)
    run_gdn(backend, pkg.gdn_forward)
    assert len(backend.lib.calls) == 2


STATE = types.SimpleNamespace(handle=1, channels=40, value_heads=2, value_dim=8, conv_kernel=4)


def gdn_args():
    return dict(qkv=floats(ROWS, 40), z=floats(ROWS, 16), a=floats(ROWS, 2), b=floats(ROWS, 2), a_log=floats(2),
                dt_bias=floats(2), conv_weight=floats(40, 4), norm=floats(8), out=floats(ROWS, 16))


def run_gdn(backend, call, **change):
    tree = [[-1, 0, 0]] if call is pkg.gdn_tree_forward else []
    call(backend, STATE, [0], [ROWS], *tree, **dict(gdn_args(), **change))


@pytest.mark.parametrize("name", list(gdn_args()))
def test_gdn_tree_refuses(backend, name):
    for how, error in ((short, ValueError), (torch.Tensor.half, TypeError)) + (
            () if name == "qkv" else ((bf16, TypeError), (on_device, ValueError))):
        with pytest.raises(error, match=name):
            run_gdn(backend, pkg.gdn_tree_forward, **{name: how(gdn_args()[name])})
    assert not backend.lib.calls


def test_gdn_tree_takes(backend):
    run_gdn(backend, pkg.gdn_tree_forward)
    run_gdn(backend, pkg.gdn_tree_forward, **{n: bf16(gdn_args()[n]) for n in ("qkv", "z", "a", "b")})
    assert len(backend.lib.calls) == 2


def test_gather(backend):
    kv = types.SimpleNamespace(handle=1, width=KVH * DIM)
    reads = [(kv, 0, 5, [1, 2, 2]), (kv, 1, 0, 4)]

    def gather(keys, values):
        pkg.kv_gather(backend, reads, keys, values)

    good = floats(7, KVH * DIM)
    for keys, values, error, text in [
            (good, bf16(good), TypeError, "values is bfloat16"),
            (bf16(good), good, TypeError, "values is float32"),
            (good.half(), good.half(), TypeError, "keys is float16"),
            (good[:6], good, ValueError, "keys has"),
            (good, short(good), ValueError, "values has"),
            (on_device(good), good, ValueError, "values is not where"),
            (good, on_device(good), ValueError, "values is not where")]:
        with pytest.raises(error, match=text):
            gather(keys, values)
    assert not backend.lib.calls
    gather(good, good.clone())
    gather(bf16(good), bf16(good))
    gather(good.numpy(), good.numpy())
    gather(np.zeros((9, KVH * DIM), np.float32), good)
    assert len(backend.lib.calls) == 4
