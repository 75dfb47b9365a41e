"""f16 attention over many keys of small weight beside one that dominates.

Weights are rounded to f16 for the product with V.  They are taken at 2^7 and
more times their size, so a rounding is off by 2^-11 of a weight, or by 2^-25 /
2^7 = 2^-32 of the largest weight where that is more (f16 below 2^-14 has a
fixed step); sum p >= the largest weight, so with V's values 0 and 1
    |out - exact| <= n 2^-32 + (2 ds + (n + 16) 2^-24 + 2 x 2^-11) out (1 + 2^-10)
(the result's own rounding is the second 2^-11), ds the bound on a score: here
(hd + 2) 2^-24 |s| + 4 x 2^-24 (2 |s| + 1), and 2^-25 for a result below 2^-14."""
import numpy as np
import pytest
import torch

from test_batch_gpu import Dev, run_prefix, say
from yule_amd import DType

pytestmark = pytest.mark.gpu

HD, TOP = 64, 18.0   # 2^-26 = e^-18.02: below the smallest step of f16


def inputs(n):
    """Scores TOP at key 0 and 0 elsewhere; V 0 at key 0 and 1 elsewhere."""
    k, v = torch.zeros(n, HD, dtype=torch.float16), torch.ones(n, HD, dtype=torch.float16)
    k[0, 0], v[0] = TOP, 0
    return k, v


def query(rows, heads):
    q = torch.zeros(rows, heads, HD, dtype=torch.float16)
    q[:, :, 0] = HD ** 0.5
    return q.view(rows, heads * HD)


def check_small(got, n):
    """got: results of rows that see n - 1 keys of weight e^-TOP beside the one."""
    n = torch.as_tensor(n, dtype=torch.float64)
    want = (n - 1) * np.exp(-TOP) / (1 + (n - 1) * np.exp(-TOP))
    ds = (HD + 2) * 2.0 ** -24 * TOP + 4 * 2.0 ** -24 * (2 * TOP + 1)
    bound = n * 2.0 ** -32 + (2 * ds + (n + 16) * 2.0 ** -24 + 2.0 ** -10) * want * (1 + 2.0 ** -10) + 2.0 ** -25
    off = (got.double() - want[:, None]).abs()
    worst = (off / bound[:, None]).max().item()
    assert worst <= 1.0, f"{worst:.2f} of the bound"


@pytest.mark.parametrize("heads,kv,lens", [(4, 1, [1700]), (16, 16, [900, 400] + [1] * 80), (32, 8, [2100])])
def test_prompt_attn_small_weights(hip, heads, kv, lens):
    """By workgroups of 32 pairs, of 128, and of 128 with split keys."""
    say(f"[batch] prompt_attn F16 {heads}/{kv}, many small weights, lens {lens[:2]}")
    n = sum(lens)
    k, v = inputs(n)
    k, v = (x[:, None].expand(n, kv, HD).reshape(n, kv * HD) for x in (k, v))
    with Dev(hip) as d:
        out = d.new(n * heads * HD * 2)
        hip.prompt_attn(d.up(query(n, heads)), d.up(k), d.up(v), out, d.up(np.cumsum([0] + lens).astype(np.uint32)), len(lens), n,
                        heads, kv, HD, DType.F16)
        got = d.down(out, (n, heads * HD), DType.F16)
    check_small(got[:lens[0]], np.arange(1, lens[0] + 1))


@pytest.mark.parametrize("heads,kv,prefix,cap,seqs", [(4, 1, 400, 100, 3), (4, 1, 16384, 0, 2), (16, 16, 16384, 0, 40)])
def test_prefix_attn_small_weights(hip, heads, kv, prefix, cap, seqs):
    """In one launch, by chunks, and by chunks that share tiles.  (Every chunk but the first has weights of 1 of its own: what
    is small is the first one's.)"""
    say(f"[batch] prefix_attn F16 {heads}/{kv}, many small weights, prefix {prefix}, tails {cap}, {seqs} sequences")
    k, v = (x[:, None].expand(prefix + cap, kv, HD).reshape(prefix + cap, kv * HD) for x in inputs(prefix + cap))
    kt, vt = (x[prefix:].repeat(seqs, 1) for x in (k, v))
    with Dev(hip) as d:
        got = run_prefix(hip, d, query(seqs, heads), k[:prefix], v[:prefix], kt, vt, [cap] * seqs, cap, 1, heads, kv, HD, DType.F16)
    check_small(got, np.full(seqs, prefix + cap))
