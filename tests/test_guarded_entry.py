"""The body of a C entry on the CPU (a host program with a stand-in for the two
device calls): exceptions become an error with a message of its own, and the
caller's device is current again afterwards."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
ROCM = Path("/opt/rocm/include")

PROGRAM = r"""
#include <cstdio>
#include <new>
#include <stdexcept>
#include "internal.h"

static int current = 2;
extern "C" hipError_t hipGetDevice(int *d) { *d = current; return hipSuccess; }
extern "C" hipError_t hipSetDevice(int d) { current = d; return hipSuccess; }
static std::string last;
namespace yule {
int set_error(int code, const std::string &m) { last = m; return code; }
int hip_error(hipError_t e, const char *) { return e == hipSuccess ? YULE_OK : YULE_ERR_HIP; }
}
using namespace yule;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    yule_hip_backend be;
    be.device = 1;
    last = "of an earlier call";
    CHECK(guarded("a", &be, []() -> int { throw std::bad_alloc(); }) == YULE_ERR_OOM && last == "out of memory" && current == 2);
    last = "of an earlier call";
    CHECK(guarded("a", &be, []() -> int { throw std::length_error("x"); }) == YULE_ERR_OOM && last == "out of memory" && current == 2);
    int seen = -1;
    CHECK(guarded("a", &be, [&]() -> int { seen = current; return 7; }) == 7 && seen == 1 && current == 2);
    CHECK(guarded("a", nullptr, []() -> int { return 0; }) == YULE_ERR_INVALID && last == "null backend");
    printf("ok\n");
    return 0;
}
"""


def test_guarded(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None or not (ROCM / "hip" / "hip_runtime.h").exists():
        pytest.skip("no g++, or no HIP headers")
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-O1", "-std=c++17", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}", f"-I{ROOT / 'yule_amd' / 'csrc'}",
                    str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t"), "-lpthread"], check=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
