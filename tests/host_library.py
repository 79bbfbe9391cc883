"""The library's host code without a GPU (host_library.cpp), loaded as the engine loads
the library."""
import ctypes as C
import importlib
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
SOURCES = ["attention", "gdn", "gdn_tree", "kv", "kv_compact", "plugin", "tree_attention"]
pkg = importlib.import_module("safetyraise-lmengine_amd")


@pytest.fixture(scope="session")
def host_path(tmp_path_factory):
    where = tmp_path_factory.mktemp("host_library")
    csrc = ROOT / "safetyraise-lmengine_amd" / "csrc"
    flags = ["-std=c++17", "-O1", "-g", "-fPIC", "-fno-builtin-memcpy", "-Wall", "-D__HIP_PLATFORM_AMD__",
             "-I/opt/rocm/include", f"-I{ROOT / 'include'}", f"-I{csrc}"]
    jobs = [(subprocess.Popen(["g++", *flags, "-c", str(src), "-o", str(where / (src.stem + ".o"))]), src)
            for src in [csrc / f"{s}.cpp" for s in SOURCES] + [ROOT / "tests" / "host_library.cpp"]]
    for job, src in jobs:
        assert job.wait() == 0, src
    path = where / "libhost.so"
    subprocess.run(["g++", "-shared", "-Wl,--wrap=memcpy", "-Wl,-Bsymbolic", "-o", str(path),
                    *[str(where / (src.stem + ".o")) for _, src in jobs]], check=True)
    return path


@pytest.fixture
def host(host_path):
    """A backend on the host library; .test: its functions for tests."""
    backend = pkg.NativeBackend.load(host_path)
    test = backend.test = C.CDLL(str(host_path))
    test.test_seed.argtypes = [C.c_uint64]
    test.test_fail.argtypes = [C.c_char_p, C.c_int]
    test.test_pool.argtypes = [C.c_void_p]
    test.test_free_pages.argtypes = [C.c_void_p]
    test.test_free_pages.restype = C.c_uint64
    test.test_fail(b"", 0)
    yield backend
    backend.close()
