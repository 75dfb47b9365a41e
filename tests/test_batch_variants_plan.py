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
