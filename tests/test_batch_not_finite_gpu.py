"""Values that are infinite or NaN and that rows do see: they reach the dims
that they stand in, and no others."""
import numpy as np
import pytest
import torch

from test_batch_gpu import TYPES, Dev, check, normal, prefix_inputs, prefix_reference, prompt_reference, run_prefix, say
from yule_amd import DType

pytestmark = pytest.mark.gpu


def same_value(got, bad):
    return torch.isnan(got).all() if bad != bad else (got.float() == bad).all()


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("hd", [8, 40, 64, 80, 136, 200])
def test_prompt_attn_seen_not_finite(hip, dt, bad, hd):
    """One value of V that every later row sees, in the last dims of a head that does not fill its padded size: the head's
    other dims, and the rows before, are the ones of V without it."""
    heads, kv, n, at, dim = 2, 1, 300, 5, hd - 3
    say(f"[batch] prompt_attn {dt.name} x{hd}, {bad} in a row that is seen")
    q, k, v = normal(1, (n, heads * hd), dt, 1.5), normal(2, (n, kv * hd), dt), normal(3, (n, kv * hd), dt)
    v[at, dim] = 0
    want, bound = prompt_reference(q, k, v, [n], heads, kv, hd, dt)
    v[at, dim] = bad
    with Dev(hip) as d:
        out = d.new(q.numel() * q.element_size())
        hip.prompt_attn(d.up(q), d.up(k), d.up(v), out, d.up(np.array([0, n], np.uint32)), 1, n, heads, kv, hd, dt)
        got = d.down(out, tuple(q.shape), dt)
    has = torch.zeros(q.shape, dtype=torch.bool)
    has[at:, dim::hd] = True
    assert same_value(got[has], bad)
    check(got[~has], want[~has], bound[~has], "the others")


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("hd,prefix", [(40, 90), (80, 420), (80, 1500)])
def test_prefix_attn_seen_not_finite(hip, dt, bad, hd, prefix):
    heads, kv, cap, lens, tokens, at, dim = 4, 2, 20, [20, 7], 2, 5, hd - 1
    say(f"[batch] prefix_attn {dt.name} x{hd}, prefix {prefix}, {bad} in a row that is seen")
    q, kp, vp, kt, vt = prefix_inputs(10, heads, kv, hd, prefix, cap, lens, tokens, dt)
    vp[at, dim] = 0   # of KV head 0
    want, bound = prefix_reference(q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    vp[at, dim] = bad
    with Dev(hip) as d:
        got = run_prefix(hip, d, q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    has = torch.zeros(q.shape, dtype=torch.bool)
    has[:, dim:heads // kv * hd:hd] = True
    assert same_value(got[has], bad)
    check(got[~has], want[~has], bound[~has], "the others")


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("n", [3, 700])
def test_scores_of_minus_infinity(hip, dt, n):
    """Keys whose scores are minus infinity weigh nothing; a row that has no others gives zeros."""
    say(f"[batch] prompt_attn and prefix_attn {dt.name}, {n} rows, scores of minus infinity")
    heads, kv, hd, none = 2, 1, 64, 2
    q, k, v = normal(1, (n, heads * hd), dt).abs(), normal(2, (n, hd), dt), normal(3, (n, hd), dt)
    q = q + 0.5                                   # positive: q . k is minus infinity where k is in one dim
    want, bound = prompt_reference(q[none:], k[none:], v[none:], [n - none], heads, kv, hd, dt)
    k[:none, 5] = -float("inf")
    with Dev(hip) as d:
        out = d.new(q.numel() * q.element_size())
        args = d.up(q), d.up(k), d.up(v)
        hip.prompt_attn(*args, out, d.up(np.array([0, n], np.uint32)), 1, n, heads, kv, hd, dt)
        got = d.down(out, tuple(q.shape), dt)
        last = run_prefix(hip, d, q[-1:], k, v, k[:0], v[:0], [0], 0, 1, heads, kv, hd, dt)
        first = run_prefix(hip, d, q[-1:], k[:none], v[:none], k[:0], v[:0], [0], 0, 1, heads, kv, hd, dt)
    assert (got[:none] == 0).all() and (first == 0).all()
    check(got[none:], want, bound, "prompt_attn")
    check(last, want[-1:], bound[-1:], "prefix_attn")
