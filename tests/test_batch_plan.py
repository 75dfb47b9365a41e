"""The batched serving operators' host-checkable rules on the CPU: refusals of
row layouts and head shapes, and that what prefix_attn's plan places lies
inside its workspace and covers every key once (a small host program over
batch_plan.h); the copies into LDS keep their wait state."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "yule_amd" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "batch_plan.h"
using namespace yule;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    // rows: offset, stride, rows, width, element bytes, buffer bytes, alignment
    CHECK(!check_rows(0, 64, 10, 64, 4, 2560, 16));
    CHECK(check_rows(0, 64, 10, 64, 4, 2559, 16));            // one byte short
    CHECK(check_rows(4, 64, 10, 64, 4, 2560, 16));            // past the end by the offset
    CHECK(!check_rows(64, 64, 9, 64, 4, 2560, 16));
    CHECK(check_rows(0, 60, 10, 64, 4, 1 << 20, 16));         // overlapping rows
    CHECK(check_rows(2, 64, 10, 64, 4, 1 << 20, 16));         // not aligned
    CHECK(check_rows(0, 66, 10, 64, 4, 1 << 20, 16));
    CHECK(!check_rows(1, 65, 10, 64, 4, 1 << 20, 4));
    CHECK(!check_rows(0, 0, 1, 64, 4, 256, 16));              // one row: any stride
    CHECK(!check_rows(0, 0, 0, 64, 4, 0, 16));                // none
    CHECK(check_rows(0, 1u << 24, 2, 64, 4, ~0ull, 16));      // stride too long
    CHECK(!check_rows(0, (1u << 24) - 4, 1ull << 37, 64, 4, ~0ull, 16));
    CHECK(check_rows(~0ull - 3, 64, 2, 64, 4, 1 << 20, 16));  // sums that wrap
    CHECK(check_rows(0, 64, ~0ull, 64, 4, 1 << 20, 16));
    CHECK(check_rows(0, ~0ull, 2, 64, 4, 1 << 20, 16));
    CHECK(check_rows(0, 64, 2, ~0ull, 4, 1 << 20, 16));
    CHECK(!check_heads(32, 4, 64) && !check_heads(1, 1, 8) && !check_heads(12, 2, 256));
    CHECK(check_heads(32, 5, 64) && check_heads(0, 1, 64) && check_heads(4, 0, 64) && check_heads(4, 8, 64));
    CHECK(check_heads(4, 4, 0) && check_heads(4, 4, 12) && check_heads(4, 4, 264) && check_heads(8192, 8, 64));
    CHECK(attn_elem_bytes(YULE_DTYPE_F32) == 4 && attn_elem_bytes(YULE_DTYPE_F16) == 2 &&
          attn_elem_bytes(YULE_DTYPE_BF16) == 2 && attn_elem_bytes(YULE_DTYPE_Q8_0) == 0);
    for (uint32_t hd = 8; hd <= 256; hd += 8) {
        const uint32_t d4 = attn_padded_dim(hd, 4), d2 = attn_padded_dim(hd, 2);
        CHECK(d4 >= hd && d4 % 32 == 0 && d4 - hd < 32);   // f32: some of the head in every piece of 32 dims
        CHECK(d2 >= hd && (d2 == 64 || d2 == 96 || d2 == 128 || d2 == 256));
    }
    // prompts: the tiles of any split into sequences fit, and the shapes of the GPU tests take the kernel they are for
    for (int i = 0; i < 20000; i++) {
        const uint32_t kv = 1 + (i * 7919u >> 3) % 16, group = 1 + (i * 104729u >> 4) % 16, hd = 8 * (1 + i % 32);
        const uint32_t seqs = 1 + (i * 31u) % 100;
        uint64_t rows = 0, tiles32 = 0, tiles128 = 0;
        for (uint32_t s = 0; s < seqs; s++) {
            const uint32_t n = (i * 13u + s * 977u) % 1500;
            rows += n;
            tiles32 += ((uint64_t)n * group + 31) / 32;
            tiles128 += ((uint64_t)n * group + 127) / 128;
        }
        for (uint32_t elem = 2; elem <= 4; elem += 2) {
            const PromptPlan p = prompt_plan(seqs, (uint32_t)rows, kv * group, kv, hd, elem, 256);
            CHECK((p.slots == 32 && p.tiles >= tiles32) || (p.slots == 128 && p.tiles >= tiles128));
            CHECK(p.split == 1 || (p.split == 2 && p.slots == 128 && hd <= 128));
            CHECK(elem == 2 || p.slots == 32);
        }
    }
    CHECK(attn_block_room(64, 2) == 4 && attn_block_room(80, 2) == 3 && attn_block_room(128, 2) == 2 && attn_block_room(256, 2) == 1);
    CHECK(prompt_plan(2, 24, 8, 1, 64, 2, 256).slots == 32);
    CHECK(prompt_plan(72, 1000, 16, 16, 64, 2, 256).slots == 128 && prompt_plan(72, 1000, 16, 16, 64, 2, 256).split == 1);
    CHECK(prompt_plan(72, 1000, 32, 16, 256, 2, 256).slots == 128 && prompt_plan(72, 1000, 32, 16, 80, 2, 256).slots == 128);
    CHECK(prompt_plan(1, 1100, 32, 8, 128, 2, 256).split == 2 && prompt_plan(2, 1100, 32, 8, 128, 2, 256).split == 2);
    CHECK(prompt_plan(1, 1100, 64, 16, 40, 2, 256).split == 1);
    // plans: chunks cover the keys once, jobs fit, results lie in the workspace
    unsigned seed = 1;
    auto rnd = [&](uint32_t n) { seed = seed * 1664525u + 1013904223u; return (seed >> 8) % n; };
    for (int i = 0; i < 20000; i++) {
        const uint32_t kv = 1 + rnd(16), group = 1 + rnd(16), hd = 8 * (1 + rnd(32)), seqs = 1 + rnd(200);
        const uint32_t tokens = 1 + rnd(64), prefix = rnd(3) ? rnd(1u << (1 + rnd(20))) : 0;
        const uint32_t cap = rnd(5) ? rnd(1u << (1 + rnd(14))) : 0;
        const PrefixPlan p = prefix_plan(prefix, cap, seqs, tokens, kv * group, kv, hd, 2 + 2 * rnd(2), 256);
        CHECK(p.rows == (uint64_t)seqs * tokens * kv * group);
        CHECK((uint64_t)p.p_chunk * p.n_p >= prefix && (!p.n_p || (uint64_t)p.p_chunk * (p.n_p - 1) < prefix));
        CHECK((uint64_t)p.t_chunk * p.n_t >= cap && (!p.n_t || (uint64_t)p.t_chunk * (p.n_t - 1) < cap));
        CHECK(p.n_p + p.n_t <= kMaxParts);
        CHECK((prefix == 0) == (p.n_p == 0) && (cap == 0) == (p.n_t == 0));
        CHECK((uint64_t)p.p_tiles * p.p_slots >= (uint64_t)seqs * tokens * group && p.p_slots % 32 == 0);
        CHECK((uint64_t)p.t_tiles * kAttnTileRows >= (uint64_t)tokens * group);
        CHECK(p.p_jobs == (uint64_t)p.n_p * p.p_tiles * kv && p.t_jobs == (uint64_t)p.n_t * p.t_tiles * kv * seqs);
        if (p.n_p + p.n_t) {
            const uint64_t last = (uint64_t)(p.n_p + p.n_t - 1) * p.rows + p.rows - 1;   // the last chunk's last row
            CHECK((last + 1) * 8 <= p.ml_bytes && p.ml_bytes % 256 == 0 && (last + 1) * hd * 4 <= p.o_bytes);
            CHECK(p.ml_bytes + p.o_bytes == p.bytes());
        }
    }
    // the shapes of the GPU tests take both ways
    CHECK(prefix_plan(33, 20, 3, 1, 8, 2, 64, 2, 256).direct && prefix_plan(33, 20, 3, 1, 8, 2, 64, 4, 256).direct);
    CHECK(!prefix_plan(300, 70, 4, 5, 6, 2, 80, 4, 256).direct && prefix_plan(300, 70, 4, 5, 6, 2, 80, 2, 256).direct);
    CHECK(!prefix_plan(520, 600, 4, 1, 2, 2, 8, 2, 256).direct && !prefix_plan(1333, 90, 40, 1, 8, 2, 128, 2, 256).direct);
    CHECK(!prefix_plan(600, 40, 3, 4, 4, 2, 64, 2, 256).direct && !prefix_plan(600, 40, 3, 4, 4, 2, 64, 4, 256).direct);
    printf("ok\n");
    return 0;
}
"""


def test_refusals_and_plans(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    subprocess.run([gxx, "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_copies_into_lds_wait_after_m0():
    text = (CSRC / "batch_attn.hip").read_text()
    copies = re.findall(r'"s_mov_b32 m0, [^"]*"', text)
    assert copies and all(re.search(r"m0, %\d\\n\\ts_nop 0\\n\\tglobal_load_lds_dwordx4", c) for c in copies)


def test_null_backend_is_refused():
    """The entries turn a null backend into an error before anything else."""
    import ctypes as C

    from yule_amd.backend import Rows, load_library
    lib = load_library()
    r = C.byref(Rows(1, 64))
    assert lib.yule_hip_prompt_attn(None, r, r, r, r, 1, 1, 1, 1, 1, 64, 0) == 1
    assert lib.yule_hip_prefix_attn(None, r, r, r, 1, r, r, 1, 1, r, 1, 1, 1, 1, 64, 0) == 1
    assert lib.yule_hip_verify_drafts(None, r, r, 1, 1, 0, 1, 1, 1, 1, 64) == 1
    assert b"null backend" in lib.yule_hip_last_error()
