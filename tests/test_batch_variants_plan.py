"""Which kernels the shapes of the GPU tests take (a small host program over
batch_plan.h), so that every variant that a call can reach is run by a test."""
import shutil
import subprocess
from pathlib import Path

import pytest

import batch_shapes

CSRC = Path(__file__).resolve().parent.parent / "yule_amd" / "csrc"
CUS = 256   # of an MI355X

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "batch_plan.h"
using namespace yule;
int main(int argc, char **argv) {
    auto u = [&](int i) { return (uint32_t)strtoul(argv[i], nullptr, 10); };
    if (argc == 8) {   // sequences, rows, heads, KV heads, head_dim, element bytes, CUs
        const PromptPlan p = prompt_plan(u(1), u(2), u(3), u(4), u(5), u(6), u(7));
        printf("%u %u\n", p.slots, p.split);
    } else {           // prefix, tail, sequences, tokens, heads, KV heads, head_dim, element bytes, CUs
        const PrefixPlan p = prefix_plan(u(1), u(2), u(3), u(4), u(5), u(6), u(7), u(8), u(9));
        printf("%d %u %u\n", (int)p.direct, p.p_slots, p.n_p + p.n_t);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("plan")
    (d / "t.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-O1", "-std=c++17", "-Wall", f"-I{CSRC}", str(d / "t.cpp"), "-o", str(d / "t")], check=True)

    def ask(*args):
        r = subprocess.run([str(d / "t"), *map(str, args)], capture_output=True, text=True, timeout=60, check=True)
        return [int(x) for x in r.stdout.split()]

    return ask


def elem(dt):
    return 4 if dt == batch_shapes.F32 else 2


@pytest.mark.parametrize("dt,heads,kv,hd,lens,slots,split", batch_shapes.PROMPTS)
def test_prompt_shapes(plan, dt, heads, kv, hd, lens, slots, split):
    assert plan(len(lens), sum(lens), heads, kv, hd, elem(dt), CUS) == [slots, split]


@pytest.mark.parametrize("heads,kv,hd,prefix,cap,lens,tokens", batch_shapes.SHORT)
def test_short_shapes(plan, heads, kv, hd, prefix, cap, lens, tokens):
    for dt in (batch_shapes.F32, batch_shapes.F16):
        assert plan(prefix, cap, len(lens), tokens, heads, kv, hd, elem(dt), CUS)[0] == 1


@pytest.mark.parametrize("shape,join,p_slots", batch_shapes.PREFIXES)
def test_prefix_shapes(plan, shape, join, p_slots):
    heads, kv, hd, prefix, cap, lens, tokens = shape
    for dt, want in p_slots.items():
        direct, got, parts = plan(prefix, cap, len(lens), tokens, heads, kv, hd, elem(dt), CUS)
        assert not direct and got == want
        # the join's rule, as its launch has it
        lanes = 16 if hd <= 64 else 32 if hd <= 128 else 64
        threads, ahead = (64, 0) if parts <= 2 * 64 // lanes else (256, 0) if parts <= 4 * 256 // lanes else (256, 8)
        assert (threads, lanes, ahead) == join, (dt, parts)


ROWS = r"""
#include <cstdio>
#include <initializer_list>
#include "batch_plan.h"
using namespace yule;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    const uint64_t big = 1ull << 45, far = 1ull << 24;
    // one row: its stride is never looked at
    CHECK(!check_rows(0, far, 1, 64, 4, big, 16) && !check_rows(8, ~0ull, 1, 64, 2, big, 16));
    CHECK(!check_rows(0, far - 4, 2, 64, 4, big, 16) && check_rows(0, far, 2, 64, 4, big, 16));   // attention's limit
    // rows of probabilities: any stride, a vocabulary's of 2^24 and more among them, inside the buffer
    for (uint64_t n = 1; n <= 4; n++)
        for (uint64_t vocab : {far - 1, far, far + 5, (uint64_t)kMaxVocab}) {
            CHECK(!check_rows(0, vocab, n, vocab, 4, 4 * n * vocab, 4, kAnyStride));
            CHECK(check_rows(0, vocab, n, vocab, 4, 4 * n * vocab - 4, 4, kAnyStride));
            CHECK(check_rows(1, vocab, n, vocab, 4, 4 * n * vocab, 4, kAnyStride));
        }
    CHECK(check_rows(0, ~0ull, 2, 64, 4, big, 4, kAnyStride) && check_rows(0, 1ull << 62, 2, 64, 4, big, 4, kAnyStride));
    printf("ok\n");
    return 0;
}
"""


def test_strides(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    (tmp_path / "t.cpp").write_text(ROWS)
    subprocess.run([gxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
