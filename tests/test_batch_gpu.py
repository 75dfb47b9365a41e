"""The batched serving operators on the GPU against plain 64-bit references:
prompt_attn, prefix_attn and verify_drafts, at the sizes, layouts and masks
where they can go wrong, their refusals, and a run of them together.

Tolerances.  u = 2^-24 (f32).  A score is a sum of hd products in f32 in some
order: off by at most (hd + 2) u scale sum |q||k| with the multiplication by the
scale; the exponent's fused multiply-add and 2^x add at most 4 u (|s| + |m| + 1)
more.  With ds the bound on a score, a weight is off by a factor 1 +- 2 ds (its
own and the sum's), the f32 sums over n keys and the joins add (n + 16) u:
    |out - exact| <= (2 ds + (n + 16) u) sum p |v|.
16-bit types round each weight to the type for the product with V: eps / 2 of
it, eps of the type (f16 below 2^-14: 2^-25), and the result once more.
"""
import sys
import threading

import numpy as np
import pytest
import torch

from yule_amd import DType, synth
from yule_amd.backend import NO_TOKEN, HipBackend, Rows, YuleGpuError

pytestmark = pytest.mark.gpu

TYPES = {DType.F32: torch.float32, DType.F16: torch.float16, DType.BF16: torch.bfloat16}
U = 2.0 ** -24


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def normal(seed, shape, dt, scale=1.0):
    return torch.from_numpy(synth.gauss(seed, shape)).mul(scale).to(TYPES[dt])


def bits(t):
    return t.contiguous().view(torch.int16).numpy() if t.element_size() == 2 else t.contiguous().numpy()


class Dev:
    """Buffers of one test, freed at its end."""

    def __init__(self, hip):
        self.hip, self.h = hip, []

    def up(self, t):
        a = bits(t) if isinstance(t, torch.Tensor) else np.ascontiguousarray(t)
        self.h.append(self.hip.upload(a) if a.size else self.hip.allocate(16))
        return self.h[-1]

    def new(self, n_bytes):
        self.h.append(self.hip.allocate(n_bytes))
        return self.h[-1]

    def down(self, h, shape, dt):
        if dt == DType.F32:
            return torch.from_numpy(self.hip.download(h, shape))
        return torch.from_numpy(self.hip.download(h, shape, np.int16)).view(TYPES[dt])

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for h in self.h:
            self.hip.free(h)


def attend(q, k, v, dt):
    """(result, bound) in f64 of one query row over its visible keys: q [hd], k, v [n, hd]."""
    q, k, v = q.double(), k.double(), v.double()
    if not k.shape[0]:
        return torch.zeros_like(q), torch.zeros_like(q)
    scale = q.shape[0] ** -0.5
    s = (k @ q) * scale
    p = torch.softmax(s, 0)
    ds = (q.shape[0] + 2) * U * scale * (k.abs() @ q.abs()).max() + 4 * U * (2 * s.abs().max() + 1)
    pv = p @ v.abs()
    out = p @ v
    bound = (2 * ds + (k.shape[0] + 16) * U) * pv
    if dt != DType.F32:
        eps = torch.finfo(TYPES[dt]).eps
        bound = (bound + eps / 2 * pv) * (1 + eps) + eps / 2 * out.abs()
        if dt == DType.F16:
            bound = bound + 2.0 ** -25 * (v.abs().sum(0) + 1)
    return out, bound + 1e-37


def check(got, want, bound, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    share = torch.where(off == 0, 0.0, off / bound)   # (rows that see nothing: 0, with a bound of 0)
    worst = share.max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound at {torch.argmax(share).item()}"
    return worst


# ---------------------------------------------------------------- packed prompts
def prompt_reference(q, k, v, lens, heads, kv, hd, dt, rows=None):
    want, bound, at, group = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0, heads // kv
    for n in lens:
        for r in range(n):
            if rows is not None and at + r not in rows:
                continue
            for h in range(heads):
                c, g = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
                want[at + r, c], bound[at + r, c] = attend(q[at + r, c], k[at:at + r + 1, g], v[at:at + r + 1, g], dt)
        at += n
    return want, bound


PROMPTS = [
    # heads, KV heads, head_dim, lengths, rows behind the last sequence
    (4, 2, 64, [1], 0),
    (8, 1, 64, [3, 0, 5, 1], 2),
    (6, 2, 80, [33, 64, 7], 0),
    (4, 4, 128, [65, 31, 32], 5),
    (2, 2, 256, [40, 3], 1),
    (3, 1, 8, [129, 2], 0),
    (4, 1, 96, [130], 0),
    (2, 1, 32, [70, 9], 0),
    (2, 1, 136, [50, 4], 2),
    (1, 1, 168, [35], 0),
    (2, 2, 200, [33, 1], 0),
    (32, 4, 64, [17, 100], 0),
]


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("heads,kv,hd,lens,spare", PROMPTS)
@pytest.mark.parametrize("fused", [False, True], ids=["apart", "fused"])
def test_prompt_attn(hip, dt, heads, kv, hd, lens, spare, fused):
    say(f"[batch] prompt_attn {dt.name} {heads}/{kv}x{hd} lens {lens} spare {spare} fused {fused}")
    qd, kvd, n = heads * hd, kv * hd, sum(lens) + spare
    q, k, v = normal(1, (n, qd), dt, 1.5), normal(2, (n, kvd), dt), normal(3, (n, kvd), dt)
    before = normal(4, (n, qd), dt)
    off = np.cumsum([0] + lens).astype(np.uint32)
    with Dev(hip) as d:
        out, offs = d.up(before), d.up(off)
        if fused:
            ld = qd + 2 * kvd
            h = d.up(torch.cat([q, k, v], 1))
            args = (Rows(h, ld), Rows(h, ld, qd), Rows(h, ld, qd + kvd))
        else:
            args = (d.up(q), d.up(k), d.up(v))
        hip.prompt_attn(*args, out, offs, len(lens), n, heads, kv, hd, dt)
        got = d.down(out, (n, qd), dt)
        hip.prompt_attn(*args, out, offs, len(lens), n, heads, kv, hd, dt)
        assert torch.equal(bits_of(got), bits_of(d.down(out, (n, qd), dt))), "not the same twice"
    total = sum(lens)
    assert torch.equal(bits_of(got[total:]), bits_of(before[total:])), "rows behind the last sequence"
    want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt)
    check(got[:total], want[:total], bound[:total], "prompt_attn")


def bits_of(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
def test_prompt_attn_long(hip, dt):
    """Many tiles, many sequences (more than a wave's lanes of them), and one row's worth of large scores."""
    heads, kv, hd = 4, 1, 64
    lens = [1, 2, 0] * 30 + [700, 257]
    n = sum(lens)
    say(f"[batch] prompt_attn {dt.name}, {len(lens)} sequences, {n} rows")
    q, k, v = normal(5, (n, heads * hd), dt), normal(6, (n, kv * hd), dt), normal(7, (n, kv * hd), dt)
    q[100] *= 40   # a softmax that is one key's
    at = n - 957
    rows = {0, 1, 2, 89, 90, at, at + 31, at + 32, at + 99, 100, at + 699, at + 700, n - 1}
    with Dev(hip) as d:
        out, offs = d.new(q.numel() * q.element_size()), d.up(np.cumsum([0] + lens).astype(np.uint32))
        hip.prompt_attn(d.up(q), d.up(k), d.up(v), out, offs, len(lens), n, heads, kv, hd, dt)
        got = d.down(out, tuple(q.shape), dt)
    want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt, rows)
    for r in sorted(rows):
        check(got[r], want[r], bound[r], f"row {r}")


# 16-bit prompts by workgroups of 128 pairs: many sequences of every length up to a few tiles, with heads that do and do
# not fill the kernels' rows, and few long ones (split over two groups of waves); tests/test_batch_plan.py has the shapes'
# plans
@pytest.mark.parametrize("dt", [DType.F16, DType.BF16], ids=lambda d: d.name)
@pytest.mark.parametrize("heads,kv,hd,lens,spare", [
    (16, 16, 64, [0, 1, 2, 63, 64, 65, 127, 128, 129] + [3] * 60 + [33, 31, 50], 4),
    (32, 16, 80, [0, 1, 31, 32, 33, 63, 64, 65, 96, 127] + [5] * 60 + [130, 20], 0),
    (32, 16, 128, [1, 64, 66, 190, 200] + [7] * 65 + [34, 0], 3),
    (32, 16, 256, [1, 40, 65] + [4] * 67 + [100, 0], 1),
    (48, 16, 96, [1, 43, 65, 129] + [4] * 67 + [100], 0),
    (32, 8, 128, [1100], 0),
    (32, 8, 120, [577, 523], 9),
    (12, 2, 80, [3000], 0),
    (64, 16, 40, [1100], 0),
])
@pytest.mark.parametrize("fused", [False, True], ids=["apart", "fused"])
def test_prompt_attn_tiles(hip, dt, heads, kv, hd, lens, spare, fused):
    n, qd, kvd = sum(lens) + spare, heads * hd, kv * hd
    say(f"[batch] prompt_attn {dt.name} {heads}/{kv}x{hd}, {len(lens)} sequences, {n} rows, fused {fused}")
    q, k, v = normal(21, (n, qd), dt, 1.5), normal(22, (n, kvd), dt), normal(23, (n, kvd), dt)
    before = normal(24, (n, qd), dt)
    with Dev(hip) as d:
        out, offs = d.up(before), d.up(np.cumsum([0] + lens).astype(np.uint32))
        if fused:
            h, ld = d.up(torch.cat([q, k, v], 1)), qd + 2 * kvd
            args = (Rows(h, ld), Rows(h, ld, qd), Rows(h, ld, qd + kvd))
        else:
            args = (d.up(q), d.up(k), d.up(v))
        hip.prompt_attn(*args, out, offs, len(lens), n, heads, kv, hd, dt)
        got = d.down(out, (n, qd), dt)
        hip.prompt_attn(*args, out, offs, len(lens), n, heads, kv, hd, dt)
        assert torch.equal(bits_of(got), bits_of(d.down(out, (n, qd), dt))), "not the same twice"
    total = sum(lens)
    assert torch.equal(bits_of(got[total:]), bits_of(before[total:]))
    assert torch.isfinite(got[:total].float()).all()
    # rows: every sequence's last, and some of the longer ones' around the tiles
    rows, at = set(), 0
    for m in lens:
        rows |= {at + r for r in (0, 15, 16, 31, 32, 33, 63, 64, 65, 100, 127, 128, m // 2, m - 1) if 0 <= r < m and (m > 8 or r == m - 1)}
        at += m
    rows = sorted(rows)[::max(1, len(rows) * heads // 2500)]
    want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt, set(rows))
    check(got[rows], want[rows], bound[rows], "prompt_attn")


@pytest.mark.parametrize("dt", [DType.F16, DType.BF16], ids=lambda d: d.name)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv,hd,lens", [(16, 16, 64, [150, 70] + [1] * 80), (32, 8, 128, [1100])])
def test_prompt_attn_tiles_hidden_not_finite(hip, dt, bad, heads, kv, hd, lens):
    say(f"[batch] prompt_attn {dt.name} {heads}/{kv}x{hd}, {bad} in hidden rows of shared tiles")
    n, at = sum(lens), 101   # of the first sequence
    q, k, v = (normal(25 + i, (n, w * hd), dt) for i, w in enumerate((heads, kv, kv)))
    rows = {0, 30, 63, 64, 90, 99, 100, lens[0] + 5 if len(lens) > 1 else 10}
    want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt, rows)
    v[at], k[at + 3] = bad, bad
    if len(lens) > 1:
        v[lens[0] - 1], v[lens[0] + 60] = bad, bad
    with Dev(hip) as d:
        out = d.new(q.numel() * 2)
        hip.prompt_attn(d.up(q), d.up(k), d.up(v), out, d.up(np.cumsum([0] + lens).astype(np.uint32)), len(lens), n, heads, kv, hd, dt)
        got = d.down(out, tuple(q.shape), dt)
    rows = sorted(rows)
    check(got[rows], want[rows], bound[rows], "rows that do not see them")
    seen = got[at:at + 3].float()
    assert (seen == bad).all() if bad == bad else torch.isnan(seen).all()
    assert not torch.isfinite(got[lens[0] - 1].float()).any()


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_prompt_attn_hidden_not_finite(hip, dt, bad):
    """What a row does not see has no influence on it, be it NaN or infinite: later rows of its sequence, other sequences,
    rows behind the last."""
    heads, kv, hd, lens, spare = 4, 2, 80, [50, 21], 3
    say(f"[batch] prompt_attn {dt.name}, {bad} in hidden rows")
    n = sum(lens) + spare
    q, k, v = normal(8, (n, heads * hd), dt), normal(9, (n, kv * hd), dt), normal(10, (n, kv * hd), dt)
    want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt)
    v[40] = bad                    # V of row 40: rows 0..39 of sequence 0 must not see it
    k[45, 3] = bad                 # K of row 45
    k[70], v[70] = bad, bad        # the last row of sequence 1
    k[71:], v[71:] = bad, bad      # behind the last sequence
    with Dev(hip) as d:
        out, offs = d.new(q.numel() * q.element_size()), d.up(np.cumsum([0] + lens).astype(np.uint32))
        hip.prompt_attn(d.up(q), d.up(k), d.up(v), out, offs, len(lens), n, heads, kv, hd, dt)
        got = d.down(out, tuple(q.shape), dt)
    check(got[:40], want[:40], bound[:40], "rows before")
    check(got[50:70], want[50:70], bound[50:70], "the other sequence")
    # and who sees it has it: V's value reaches rows 40..44 of every head
    assert (got[40:45].float() == bad).all() if bad == bad else torch.isnan(got[40:45].float()).all()


def test_prompt_attn_bad_offsets_stay_inside(hip):
    """Offsets past the rows or decreasing: nothing outside the buffers, rows of no sequence as they were."""
    heads, kv, hd, n = 2, 1, 64, 40
    say("[batch] prompt_attn, offsets out of order and range")
    q, k, v = (normal(11 + i, (n, w * hd), DType.F32) for i, w in enumerate((heads, kv, kv)))
    before = normal(20, (n, heads * hd), DType.F32)
    with Dev(hip) as d:
        args = d.up(q), d.up(k), d.up(v)
        out, offs = d.up(before), d.up(np.array([10, 5, 5, 2 ** 32 - 1, 2 ** 31], np.uint32))
        hip.prompt_attn(*args, out, offs, 4, n, heads, kv, hd)
        got = d.down(out, (n, heads * hd), DType.F32)
    assert torch.equal(got[:5], before[:5])
    want, bound = prompt_reference(q[5:], k[5:], v[5:], [35], heads, kv, hd, DType.F32)
    check(got[5:], want, bound, "rows 5..39 as one sequence")


# ---------------------------------------------------------------- shared prefix
def prefix_reference(q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt):
    want, bound, group = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), heads // kv
    for s, n in enumerate(lens):
        n = min(n, cap)
        for i in range(tokens):
            sees = max(0, n - tokens + 1 + i)
            for h in range(heads):
                c, g = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
                k = torch.cat([kp[:, g], kt[s * cap:s * cap + sees, g]])
                v = torch.cat([vp[:, g], vt[s * cap:s * cap + sees, g]])
                r = s * tokens + i
                want[r, c], bound[r, c] = attend(q[r, c], k, v, dt)
    return want, bound


PREFIXES = [
    # heads, KV heads, head_dim, prefix, tail capacity, tail lengths, tokens
    (4, 2, 64, 1, 1, [1], 1),
    (8, 2, 64, 33, 20, [20, 1, 7], 1),
    (6, 2, 80, 300, 70, [70, 5, 0, 33], 5),
    (4, 4, 128, 129, 64, [64, 31], 2),
    (2, 1, 256, 65, 40, [40, 3], 3),
    (16, 1, 64, 40, 12, [12, 3, 9, 4, 1], 4),      # 64 slots a sequence
    (4, 1, 64, 0, 30, [30, 0, 2, 1], 3),           # no prefix: rows that see nothing
    (4, 1, 64, 77, 0, [0, 9], 2),                  # no tail at all
    (2, 2, 8, 520, 600, [600, 513, 99, 2 ** 32 - 1], 1),   # more than one chunk of each; a length above the capacity
    (2, 1, 64, 10, 80, [80, 70], 64),
    (2, 2, 152, 90, 20, [20, 7], 2),
    # (above: mostly one launch for few keys; from here on by chunks)
    (6, 2, 80, 600, 70, [70, 5, 0, 33], 5),
    (4, 4, 128, 700, 64, [64, 31], 2),
    (2, 1, 256, 565, 40, [40, 3], 3),
    (16, 1, 64, 540, 12, [12, 3, 9, 4, 1], 4),
    (4, 1, 64, 0, 530, [130, 0, 2, 529], 3),
    (4, 1, 64, 577, 0, [0, 9], 2),
    (64, 1, 64, 600, 30, [3, 30], 2),
    (4, 1, 24, 70, 33, [33, 0, 5], 1),
]


def run_prefix(hip, d, q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt):
    out = d.up(torch.full_like(q, 7.0))
    args = (d.up(q), d.up(kp), d.up(vp), kp.shape[0], d.up(kt), d.up(vt), d.up(np.array(lens, np.uint32)), cap, out,
            len(lens), tokens, heads, kv, hd, dt)
    hip.prefix_attn(*args)
    got = d.down(out, tuple(q.shape), dt)
    hip.prefix_attn(*args)
    assert torch.equal(bits_of(got), bits_of(d.down(out, tuple(q.shape), dt))), "not the same twice"
    return got


def prefix_inputs(seed, heads, kv, hd, prefix, cap, lens, tokens, dt):
    b, kvd = len(lens), kv * hd
    return (normal(seed, (b * tokens, heads * hd), dt, 1.5), normal(seed + 1, (prefix, kvd), dt),
            normal(seed + 2, (prefix, kvd), dt), normal(seed + 3, (b * cap, kvd), dt), normal(seed + 4, (b * cap, kvd), dt))


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("heads,kv,hd,prefix,cap,lens,tokens", PREFIXES)
def test_prefix_attn(hip, dt, heads, kv, hd, prefix, cap, lens, tokens):
    say(f"[batch] prefix_attn {dt.name} {heads}/{kv}x{hd} prefix {prefix} tails {lens} of {cap}, {tokens} tokens")
    x = prefix_inputs(30, heads, kv, hd, prefix, cap, lens, tokens, dt)
    with Dev(hip) as d:
        got = run_prefix(hip, d, *x, lens, cap, tokens, heads, kv, hd, dt)
    want, bound = prefix_reference(*x, lens, cap, tokens, heads, kv, hd, dt)
    check(got, want, bound, "prefix_attn")
    nothing = want.abs().sum(1) == 0
    assert (got[nothing] == 0).all()


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
def test_prefix_attn_many(hip, dt):
    """A batch of more than one query tile over a longer prefix (rows of some sequences against the reference)."""
    heads, kv, hd, prefix, cap, tokens = 8, 2, 128, 1333, 90, 1
    lens = [1 + 89 * s // 39 for s in range(40)]
    say(f"[batch] prefix_attn {dt.name}, 40 sequences over 1333 rows")
    x = prefix_inputs(40, heads, kv, hd, prefix, cap, lens, tokens, dt)
    with Dev(hip) as d:
        got = run_prefix(hip, d, *x, lens, cap, tokens, heads, kv, hd, dt)
    q, kp, vp, kt, vt = x
    for s in (0, 7, 8, 31, 32, 39):
        want, bound = prefix_reference(q[s:s + 1], kp, vp, kt[s * cap:], vt[s * cap:], lens[s:s + 1], cap, 1, heads, kv, hd, dt)
        check(got[s:s + 1], want, bound, f"sequence {s}")


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("prefix", [50, 600])
def test_prefix_attn_hidden_not_finite(hip, dt, bad, prefix):
    """Rows of a tail behind its length, another sequence's, and drafts that an earlier token does not see."""
    heads, kv, hd, cap, lens, tokens = 4, 2, 64, 40, [30, 40, 8], 4
    say(f"[batch] prefix_attn {dt.name}, prefix {prefix}, {bad} in hidden rows")
    q, kp, vp, kt, vt = prefix_inputs(50, heads, kv, hd, prefix, cap, lens, tokens, dt)
    want, bound = prefix_reference(q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    kt[30:40], vt[30:40] = bad, bad                # behind sequence 0
    kt[88:120], vt[88:120] = bad, bad              # behind sequence 2
    vt[cap + 38] = bad                             # third of sequence 1's new rows: tokens 0, 1 do not see it
    with Dev(hip) as d:
        got = run_prefix(hip, d, q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    keep = [r for r in range(12) if r not in (6, 7)]
    check(got[keep], want[keep], bound[keep], "rows that do not see them")
    assert not torch.isfinite(got[6:8].float()).any()


def test_prefix_attn_far_rows(hip):
    """A cache whose rows lie past 4 GiB of its buffer."""
    heads, kv, hd, prefix, stride = 2, 1, 64, 1030, 1 << 20
    say("[batch] prefix_attn, rows past 4 GiB")
    n = prefix - 1
    q, k, v = normal(60, (1, heads * hd), DType.F32), normal(61, (prefix, hd), DType.F32), normal(62, (prefix, hd), DType.F32)
    k[:n - 2], v[:n - 2] = 0, 0   # (fresh buffers hold zeros)
    with Dev(hip) as d:
        cache, row = d.new(4 * (n * stride + 4 * hd)), d.new(4 * 2 * hd)
        for r in range(n - 2, prefix):
            hip.copy_to_device(torch.cat([k[r], v[r]]).numpy(), row)
            hip.copy_buffer_offset(row, cache, 0, 4 * r * stride, 4 * 2 * hd)
        out, lens = d.new(4 * heads * hd), d.up(np.zeros(1, np.uint32))
        hip.prefix_attn(d.up(q), Rows(cache, stride), Rows(cache, stride, hd), prefix, None, None, lens, 0, out, 1, 1,
                        heads, kv, hd)
        got = d.down(out, (1, heads * hd), DType.F32)
    want, bound = prefix_reference(q, k, v, k[:0], v[:0], [0], 0, 1, heads, kv, hd, DType.F32)
    check(got, want, bound, "far rows")


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("prefix", [70, 520])
def test_prefix_attn_continues_prompt_attn(hip, dt, prefix):
    """The newest tokens over prefix and tail are the last rows of the whole sequences as packed prompts."""
    heads, kv, hd, cap, lens, tokens = 8, 2, 64, 33, [33, 9, 5], 5
    say(f"[batch] prefix_attn against prompt_attn {dt.name}")
    _, kp, vp, kt, vt = prefix_inputs(70, heads, kv, hd, prefix, cap, lens, tokens, dt)
    whole = [prefix + n for n in lens]
    n = sum(whole)
    q = normal(76, (n, heads * hd), dt)
    k = torch.cat([x for s, m in enumerate(lens) for x in (kp, kt[s * cap:s * cap + m])])
    v = torch.cat([x for s, m in enumerate(lens) for x in (vp, vt[s * cap:s * cap + m])])
    ends = np.cumsum(whole)
    last = torch.cat([q[e - tokens:e] for e in ends])
    with Dev(hip) as d:
        out = d.new(q.numel() * q.element_size())
        hip.prompt_attn(d.up(q), d.up(k), d.up(v), out, d.up(np.concatenate([[0], ends]).astype(np.uint32)), len(lens),
                        n, heads, kv, hd, dt)
        a = d.down(out, tuple(q.shape), dt)
        b = run_prefix(hip, d, last, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    a = torch.cat([a[e - tokens:e] for e in ends])
    _, bound = prefix_reference(last, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    check(b, a.double(), 2 * bound, "the two operators")


# ---------------------------------------------------------------- verification of drafts
def verify_reference(p, q, drafts, u, lens, vocab):
    b, n = drafts.shape
    acc, tok = np.zeros(b, np.uint32), np.full((b, n + 1), NO_TOKEN, np.uint32)
    clean = lambda w: np.where(w > 0, w, 0.0)  # noqa: E731
    for s in range(b):
        a = 0
        while a < min(lens[s], n):
            x = int(drafts[s, a])
            if x >= vocab or not float(u[s, a]) * float(q[s, a, x]) < float(p[s, a, x]):
                break
            tok[s, a] = x
            a += 1
        w = clean(p[s, a].astype(np.float64))
        if a < min(lens[s], n):
            with np.errstate(invalid="ignore"):
                rest = clean(p[s, a].astype(np.float64) - q[s, a].astype(np.float64))
            rest[~(p[s, a] == p[s, a])] = 0
            w = rest if rest.any() else w
        c = np.cumsum(w)
        past = np.nonzero(c > float(u[s, n]) * c[-1])[0]
        last = np.nonzero(w)[0]
        acc[s] = a
        tok[s, a] = past[0] if past.size else last[-1] if last.size else NO_TOKEN
    return acc, tok


def run_verify(hip, d, p, q, drafts, u, lens, vocab):
    b, n = drafts.shape
    acc, tok = d.up(np.full(b, 77, np.uint32)), d.up(np.full((b, n + 1), 77, np.uint32))
    hip.verify_drafts(d.up(p), d.up(q) if n else None, d.up(drafts) if n else None, d.up(u),
                      None if lens is None else d.up(np.asarray(lens, np.uint32)), acc, tok, b, n, vocab)
    return hip.download(acc, b, np.uint32), hip.download(tok, (b, n + 1), np.uint32)


def verify_inputs(seed, b, n, vocab):
    rng = np.random.default_rng(seed)
    logits = rng.normal(size=(b, n + 1, vocab)) * 2
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p = (p / p.sum(-1, keepdims=True)).astype(np.float32)
    e = np.exp(logits[:, :n] + rng.normal(size=(b, n, vocab)) * 0.5 - logits[:, :n].max(-1, keepdims=True))
    q = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    drafts = (q / rng.exponential(size=q.shape)).argmax(-1).astype(np.uint32) if n else np.zeros((b, 0), np.uint32)
    return p, q, drafts, rng.random((b, n + 1), np.float32)


@pytest.mark.parametrize("b,n,vocab", [(1, 0, 1), (3, 4, 1), (5, 1, 7), (9, 5, 1001), (4, 3, 4095), (4, 3, 4096), (4, 3, 4097),
                                       (6, 70, 300), (2, 2, 32000), (3, 0, 50257), (1, 1, 128256)])
@pytest.mark.parametrize("ragged", [False, True])
def test_verify_drafts(hip, b, n, vocab, ragged):
    say(f"[batch] verify_drafts {b} x {n} of {vocab}, ragged {ragged}")
    p, q, drafts, u = verify_inputs(80 + n, b, n, vocab)
    lens = [max(0, n - s % 4) if s % 5 != 4 else n + 9 for s in range(b)] if ragged else None
    with Dev(hip) as d:
        acc, tok = run_verify(hip, d, p, q, drafts, u, lens, vocab)
    wa, wt = verify_reference(p, q, drafts, u, lens or [n] * b, vocab)
    assert np.array_equal(acc, wa) and np.array_equal(tok, wt)


def test_verify_drafts_distribution(hip):
    """Tokens of a drafting model and a target over 5 values: the answer's first token has the target's distribution.
    (4096 requests: a count's standard deviation is at most 32; six of them.)"""
    say("[batch] verify_drafts, distribution")
    b, rng = 4096, np.random.default_rng(3)
    pt, qt = np.array([.4, .1, .3, .2, 0], np.float32), np.array([.1, .5, .2, .1, .1], np.float32)
    p, q = np.broadcast_to(pt, (b, 2, 5)).copy(), np.broadcast_to(qt, (b, 1, 5)).copy()
    drafts = rng.choice(5, size=(b, 1), p=qt / qt.sum()).astype(np.uint32)
    with Dev(hip) as d:
        _, tok = run_verify(hip, d, p, q, drafts, rng.random((b, 2), np.float32), None, 5)
    counts = np.bincount(tok[:, 0], minlength=5)
    assert np.all(np.abs(counts - b * pt) <= 6 * np.sqrt(b * pt * (1 - pt)) + 1e-6), counts


def test_verify_drafts_edges(hip):
    """Certain acceptance and refusal, ties, numbers at the ends of [0, 1), values that are no probabilities."""
    say("[batch] verify_drafts, edges")
    one, nan = np.float32(1 - 2.0 ** -24), np.float32("nan")
    rows = [  # p rows (2), q row, draft, u (2), kept, token after it
        ([[0, 1, 0, 0], [0, 0, 1, 0]], [0, 1, 0, 0], 1, [one, .5], 1, 2),          # p = q: kept
        ([[0, 1, 0, 0], [0, 0, 1, 0]], [1, 0, 0, 0], 0, [0, .5], 0, 1),            # p = 0: not kept, even at u = 0
        ([[0, 1, 0, 0], [0, 0, 1, 0]], [1, 0, 0, 0], 1, [one, .5], 1, 2),          # q = 0 < p
        ([[0, 0, 1, 0], [0, 0, 1, 0]], [0, 1, 0, 0], 3, [one, .5], 0, 2),          # p = q = 0: not kept
        ([[.5, .5, 0, 0], [0, 0, 1, 0]], [1, 0, 0, 0], 0, [.5, .0], 0, 1),         # u q = p: not kept
        ([[.25, .25, .25, .25], [.25, .25, .25, .25]], [1, 0, 0, 0], 0, [.125, .25], 1, 1),   # the sum has to pass u
        ([[.25, .25, .25, .25], [.25, .25, .25, .25]], [1, 0, 0, 0], 0, [.125, 0], 1, 0),
        ([[.25, .25, .25, .25], [.25, .25, .5, 0]], [1, 0, 0, 0], 0, [.125, one], 1, 2),      # last with a weight
        ([[.25, .25, .25, .25], [.5, .5, 0, 0]], [1, 0, 0, 0], 0, [.125, 1.0], 1, 1),         # u = 1: the last
        ([[nan, .5, -1, .5], [0, 1, 0, 0]], [0, 0, 0, 0], 0, [.5, 0], 0, 1),       # NaN p: not kept; NaN, negative: no weight
        ([[.5, .5, 0, 0], [nan, -1, 0, 0]], [.5, .5, 0, 0], 1, [.5, .5], 1, NO_TOKEN),        # nothing to pick from
        ([[0, 0, 0, 0], [0, 0, 0, 0]], [.5, .5, 0, 0], 1, [.5, .5], 0, NO_TOKEN),
        ([[.5, .5, 0, 0], [0, 0, 0, 1]], [.5, .5, 0, 0], 9, [.5, .75], 0, 1),      # no token: p = q leaves p itself
    ]
    p, q = np.array([r[0] for r in rows], np.float32), np.array([[r[1]] for r in rows], np.float32)
    drafts, u = np.array([[r[2]] for r in rows], np.uint32), np.array([r[3] for r in rows], np.float32)
    with Dev(hip) as d:
        acc, tok = run_verify(hip, d, p, q, drafts, u, None, 4)
    for i, r in enumerate(rows):
        assert acc[i] == r[4] and tok[i, r[4]] == r[5], (i, acc[i], tok[i])
        assert (tok[i, :r[4]] == r[2]).all() and (tok[i, r[4] + 1:] == NO_TOKEN).all()


def test_verify_drafts_strides(hip):
    """Rows of probabilities as slices of wider rows, at odd offsets."""
    say("[batch] verify_drafts, strides")
    b, n, vocab, ld = 3, 2, 5001, 5007
    p, q, drafts, u = verify_inputs(90, b, n, vocab)
    wide_p, wide_q = (np.full((x.shape[0] * x.shape[1], ld), np.float32("nan")) for x in (p, q))
    wide_p[:, 3:3 + vocab], wide_q[:, 1:1 + vocab] = p.reshape(-1, vocab), q.reshape(-1, vocab)
    with Dev(hip) as d:
        acc, tok = d.new(4 * b), d.new(4 * b * (n + 1))
        hip.verify_drafts(Rows(d.up(wide_p), ld, 3), Rows(d.up(wide_q), ld, 1), d.up(drafts), d.up(u), None, acc, tok, b, n, vocab)
        got = hip.download(acc, b, np.uint32), hip.download(tok, (b, n + 1), np.uint32)
    want = verify_reference(p, q, drafts, u, [n] * b, vocab)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


# ---------------------------------------------------------------- refusals
def test_refusals(hip):
    say("[batch] refusals")
    with Dev(hip) as d:
        q, k, v, o = (d.new(4 * 256 * 8) for _ in range(4))
        off = d.new(4 * 9)
        small = d.new(4)
        ok = lambda **kw: dict(q=q, k=k, v=v, out=o, offsets=off, n_seqs=1, n_rows=8, n_heads=4, n_kv_heads=2, head_dim=64) | kw  # noqa: E731
        hip.prompt_attn(**ok())
        for kw, code in [(dict(dtype=DType.Q8_0), 2), (dict(n_kv_heads=3), 1), (dict(n_kv_heads=0), 1), (dict(head_dim=0), 1),
                         (dict(head_dim=12), 1), (dict(head_dim=264), 1), (dict(n_rows=9), 1), (dict(n_seqs=9), 1),
                         (dict(out=q), 1), (dict(out=off), 1), (dict(q=small), 1), (dict(offsets=small), 1),
                         (dict(k=10 ** 9), 1), (dict(q=Rows(q, 128)), 1), (dict(q=Rows(q, 256, 2)), 1), (dict(q=None), 1),
                         (dict(v=Rows(v, 2 ** 24)), 1), (dict(offsets=0), 1)]:
            with pytest.raises(YuleGpuError) as e:
                hip.prompt_attn(**ok(**kw))
            assert e.value.code == code, kw
        hip.prompt_attn(**ok(n_seqs=0))
        hip.prompt_attn(**ok(n_rows=0))
        kt, vt, ln = d.new(4 * 128 * 6), d.new(4 * 128 * 6), d.new(8)
        pk = lambda **kw: dict(q=q, k_prefix=k, v_prefix=v, prefix_len=8, k_tail=kt, v_tail=vt, tail_lens=ln, tail_cap=3,  # noqa: E731
                               out=o, n_seqs=2, n_tokens=2, n_heads=4, n_kv_heads=2, head_dim=64) | kw
        hip.prefix_attn(**pk())
        for kw, code in [(dict(dtype=DType.Q4_K), 2), (dict(n_tokens=0), 1), (dict(n_tokens=65), 1), (dict(prefix_len=17), 1),
                         (dict(tail_cap=4), 1), (dict(out=kt), 1), (dict(out=q), 1), (dict(out=ln), 1), (dict(n_seqs=3), 1),
                         (dict(tail_lens=small), 1), (dict(k_prefix=None), 1), (dict(v_tail=None), 1),
                         (dict(n_heads=5), 1), (dict(prefix_len=2 ** 31), 1), (dict(k_tail=Rows(kt, 128, 2)), 1)]:
            with pytest.raises(YuleGpuError) as e:
                hip.prefix_attn(**pk(**kw))
            assert e.value.code == code, kw
        hip.prefix_attn(**pk(n_seqs=0))
        p, t, u, a = d.new(4 * 10 * 3), d.new(4 * 10 * 3), d.new(12), d.new(4)
        vk = lambda **kw: dict(target=p, draft=q, draft_tokens=k, uniforms=u, draft_lens=None, accepted=a, tokens=t, n_seqs=1,  # noqa: E731
                               n_draft=2, vocab=10) | kw
        hip.verify_drafts(**vk())
        for kw in [dict(vocab=0), dict(vocab=11), dict(n_draft=3), dict(n_draft=1025), dict(accepted=p), dict(tokens=p),
                   dict(tokens=a), dict(tokens=u), dict(accepted=t), dict(draft=None), dict(target=None), dict(draft_tokens=None),
                   dict(n_seqs=2), dict(draft_lens=10 ** 9), dict(target=Rows(p, 9))]:
            with pytest.raises(YuleGpuError) as e:
                hip.verify_drafts(**vk(**kw))
            assert e.value.code == 1, kw
        hip.verify_drafts(**vk(n_seqs=0))
        hip.synchronize()


# ---------------------------------------------------------------- graphs, threads, a run together
def test_captured_and_replayed(hip):
    """The three operators in one captured graph, replayed with other data, lengths and eager work in between; the workspace
    grows between the replays (the graph's stays)."""
    say("[batch] capture and replay")
    heads, kv, hd, prefix, cap, tokens, dt = 8, 2, 64, 900, 40, 3, DType.BF16
    lens = [40, 11, 3]
    b, n, vocab = 3, 2, 9000
    be = HipBackend(0)   # its workspace starts empty
    with Dev(be) as d:
        x = prefix_inputs(100, heads, kv, hd, prefix, cap, lens, tokens, dt)
        q, kp, vp, kt, vt = (d.up(t) for t in x)
        ln, out, pout = d.up(np.array(lens, np.uint32)), d.new(x[0].numel() * 2), d.new(x[0].numel() * 2)
        offs = d.up(np.array([0, 4, 9], np.uint32))
        p, pq, drafts, u = verify_inputs(101, b, n, vocab)
        hp, hq, hd_, hu, acc, tok = d.up(p), d.up(pq), d.up(drafts), d.up(u), d.new(4 * b), d.new(4 * b * (n + 1))

        def step():
            be.prompt_attn(q, kt, vt, pout, offs, 2, 9, heads, kv, hd, dt)
            be.prefix_attn(q, kp, vp, prefix, kt, vt, ln, cap, out, b, tokens, heads, kv, hd, dt)
            be.verify_drafts(hp, hq, hd_, hu, None, acc, tok, b, n, vocab)

        def results():
            return (bits_of(d.down(pout, tuple(x[0].shape), dt)), bits_of(d.down(out, tuple(x[0].shape), dt)),
                    be.download(acc, b, np.uint32), be.download(tok, (b, n + 1), np.uint32))

        step()
        results()
        be.capture_begin()
        step()
        be.capture_end()
        for i in range(4):
            new = prefix_inputs(110 + i, heads, kv, hd, prefix, cap, lens, tokens, dt)
            for h, t in zip((q, kp, vp, kt, vt), new):
                be.copy_to_device(bits(t), h)
            be.copy_to_device(np.array([40 - i, 11 + i, 3 + 5 * i], np.uint32), ln)
            p, pq, drafts, u = verify_inputs(120 + i, b, n, vocab)
            for h, t in zip((hp, hq, hd_, hu), (p, pq, drafts, u)):
                be.copy_to_device(t, h)
            be.capture_replay()
            got = results()
            if i == 1:   # a larger call of its own: the workspace grows
                big = prefix_inputs(130, 32, 1, 64, 5000, 8, [8] * 64, 8, dt)
                bo = d.new(big[0].numel() * 2)
                be.prefix_attn(*(d.up(t) for t in big[:3]), 5000, d.up(big[3]), d.up(big[4]), d.up(np.full(64, 8, np.uint32)), 8,
                               bo, 64, 8, 32, 1, 64, dt)
                be.synchronize()
            step()
            want = results()
            for g, w in zip(got, want):
                assert np.array_equal(np.asarray(g), np.asarray(w)), f"replay {i}"
    be.close()


def test_two_threads(hip):
    """Calls from two host threads share the workspace and do not mix."""
    say("[batch] two threads")
    heads, kv, hd, tokens, dt = 4, 2, 64, 1, DType.F32
    x = [prefix_inputs(140 + 10 * i, heads, kv, hd, 700, 30, [30, 12], tokens, dt) for i in range(2)]
    wrong = []
    with Dev(hip) as d:
        want = [run_prefix(hip, d, *x[i], [30, 12], 30, tokens, heads, kv, hd, dt) for i in range(2)]

        def work(i):
            with Dev(hip) as mine:
                for _ in range(20):
                    if not torch.equal(run_prefix(hip, mine, *x[i], [30, 12], 30, tokens, heads, kv, hd, dt), want[i]):
                        wrong.append(i)

        ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
    assert not wrong


def test_serving_step(hip):
    """A batch served as a program would: prompts behind a shared prefix through prompt_attn, then drafts scored with
    prefix_attn, logits with quantized_gemm_f32, and verify_drafts on their probabilities; against the same in 64 bits."""
    say("[batch] a serving step")
    heads, kv, hd, dt = 8, 2, 32, DType.F32
    dim, vocab, prefix, cap, n = heads * hd, 512, 100, 24, 3
    own_rows = [9, 4, 17]                       # each request's rows behind the prefix, before the step
    lens = [m + n + 1 for m in own_rows]        # with the last token and its drafts
    b, tokens = 3, n + 1
    _, kp, vp, kt, vt = prefix_inputs(160, heads, kv, hd, prefix, cap, lens, tokens, dt)
    w = synth.gen_quant(DType.Q8_0, 161, vocab, dim)
    rng = np.random.default_rng(162)
    with Dev(hip) as d:
        # the prompt pass of every request's own rows (as packed prompts)
        rows = sum(own_rows)
        qp = normal(163, (rows, dim), dt)
        kc = torch.cat([kt[s * cap:s * cap + m] for s, m in enumerate(own_rows)])
        vc = torch.cat([vt[s * cap:s * cap + m] for s, m in enumerate(own_rows)])
        po = d.new(4 * rows * dim)
        hip.prompt_attn(d.up(qp), d.up(kc), d.up(vc), po, d.up(np.cumsum([0] + own_rows).astype(np.uint32)), b, rows, heads, kv, hd)
        want, bound = prompt_reference(qp, kc, vc, own_rows, heads, kv, hd, dt)
        check(d.down(po, (rows, dim), dt), want, bound, "prompt pass")
        # the step: last token and drafts of each request
        q = normal(164, (b * tokens, dim), dt, 1.5)
        ao, lo = d.new(4 * b * tokens * dim), d.new(4 * b * tokens * vocab)
        hip.prefix_attn(d.up(q), d.up(kp), d.up(vp), prefix, d.up(kt), d.up(vt), d.up(np.array(lens, np.uint32)), cap, ao, b,
                        tokens, heads, kv, hd)
        hip.quantized_gemm_f32(d.up(w), ao, lo, b * tokens, vocab, dim, DType.Q8_0)
        logits = hip.download(lo, (b * tokens, vocab))
        want, bound = prefix_reference(q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
        check(d.down(ao, (b * tokens, dim), dt), want, bound, "step")
        import oracle
        for r in (0, b * tokens - 1):
            ref = oracle.qmv_f64(int(DType.Q8_0), w, want[r].float().numpy(), vocab, dim)
            assert np.max(np.abs(logits[r] - ref)) <= 1e-3 * np.linalg.norm(ref) / np.sqrt(vocab)
        pr = d.new(4 * vocab)
        p = np.empty((b * tokens, vocab), np.float32)
        for r in range(b * tokens):             # the framework's softmax, row by row
            hip.softmax(d.up(logits[r]), pr, vocab)
            p[r] = hip.download(pr, vocab)
        p = p.reshape(b, tokens, vocab)
        pq = np.abs(p[:, :n] + rng.normal(size=(b, n, vocab)).astype(np.float32) * p[:, :n] * np.float32(.3))
        pq = (pq / pq.sum(-1, keepdims=True)).astype(np.float32)
        drafts = (pq / rng.exponential(size=pq.shape)).argmax(-1).astype(np.uint32)
        u = rng.random((b, n + 1), np.float32)
        acc, tok = run_verify(hip, d, p, pq, drafts, u, None, vocab)
    wa, wt = verify_reference(p, pq, drafts, u, [n] * b, vocab)
    assert np.array_equal(acc, wa) and np.array_equal(tok, wt)
