"""OUTPUT_BF16 in the calls that write f32: refused before anything is launched (the
library's host code, without a GPU)."""
import ctypes as C
import importlib

import numpy as np
import pytest

from host_library import host, host_path  # noqa: F401

pkg = importlib.import_module("safetyraise-lmengine_amd")
P = pkg.plugin


held = []  # (the structs have addresses alone)


def zeros(*shape, dtype=np.float32):
    held.append(np.zeros(shape, dtype))
    return held[-1]


def attention(host, pool):
    return P._attention_args(pool, [0], [2], zeros(2, 128), zeros(2, 64), zeros(2, 64), zeros(2, 3, dtype=np.int32),
                             zeros(2, 128), 2, 1, 64, 64, 1e4, 1e-6, None, None, False, False, (0, 0, 0), True, False)


def gdn(host, pool):
    return P._gdn_args(pool, [0], [2], zeros(2, pool.channels), zeros(2, 64), zeros(2, 2), zeros(2, 2), zeros(2),
                       zeros(2), zeros(pool.channels, 4), zeros(32), zeros(2, 64), 1e-6, False)


def call(host, name, args):
    status = getattr(host.lib, "safetyraise_kernel_" + name)(host.context, C.byref(args))
    return status, host.lib.safetyraise_kernel_last_error(host.context).decode()


@pytest.mark.parametrize("name", ["attention_forward", "gdn_forward", "gdn_tree_forward"])
def test_refused(host, name):  # noqa: F811
    if name == "attention_forward":
        pool = pkg.KvCache(host, 1, 64, 16, 8, 64, 1)
    else:
        pool = pkg.GdnState(host, 1, 2, 32, 32, 4, 1, keep_rows=4)
    pool.open()
    args = whole = (attention if name == "attention_forward" else gdn)(host, pool)
    if name == "gdn_tree_forward":
        whole = P.GdnTreeArgs()
        whole.struct_size, whole.gdn, whole.parents = C.sizeof(whole), args, (C.c_int32 * 2)(-1, 0)
        args = whole.gdn
    status, text = call(host, name, whole)
    assert "OUTPUT_BF16" not in text  # (the host library launches no such kernel)
    args.flags |= pkg.OUTPUT_BF16
    status, text = call(host, name, whole)
    assert status == 1 and "OUTPUT_BF16" in text
    if name == "attention_forward":
        assert pool.len(0) == 0
    pool.destroy()
