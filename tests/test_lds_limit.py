"""LdsLimit (csrc/sr_internal.hpp): a kernel's limit is set once on every device that
launches it, without a GPU."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include "sr_internal.hpp"
static int device = 0, fails = 0;
extern "C" hipError_t hipGetDevice(int *d) { return *d = device, hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void *kernel, hipFuncAttribute, int bytes) {
    printf("%d:%d%s ", device, bytes, fails > 0 ? "!" : "");
    return fails-- > 0 ? hipErrorInvalidValue : hipSuccess;
}
int main() {
    static sr::LdsLimit limit, other;
    auto launch = [&](sr::LdsLimit &l, int d) { return device = d, l.allow(nullptr, 90000) == hipSuccess; };
    bool ok = launch(limit, 0) && launch(limit, 0) && launch(limit, 3) && launch(limit, 0) && launch(limit, 3);
    ok = ok && launch(other, 3);
    fails = 1;
    ok = ok && !launch(other, 5) && launch(other, 5) && launch(other, 5);
    ok = ok && launch(limit, 64) && launch(limit, 64) && launch(limit, 63) && launch(limit, 63);
    printf("%s\n", ok ? "ok" : "wrong");
}
"""


def test_set_once_per_device(tmp_path):
    (tmp_path / "lds.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{ROOT / 'include'}", f"-I{ROOT / 'safetyraise-lmengine_amd' / 'csrc'}",
                    str(tmp_path / "lds.cpp"), "-o", str(tmp_path / "lds")], check=True)
    out = subprocess.run([str(tmp_path / "lds")], capture_output=True, text=True, check=True).stdout.split()
    assert out == ["0:90000", "3:90000", "3:90000", "5:90000!", "5:90000", "64:90000", "64:90000", "63:90000", "ok"]
