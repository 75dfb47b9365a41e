"""The batched operators' variants that only some shapes reach: prompts by eight
waves for every head size, prefixes whose tiles the sequences share, joins of
many chunks; and verification of rows of many chunks, more than 64 of them, and
more sequences than one launch takes."""
import numpy as np
import pytest
import torch

import batch_shapes
from test_batch_gpu import (TYPES, Dev, check, normal, prefix_inputs, prefix_reference, prompt_reference, run_prefix, run_verify,
                            say, verify_reference)
from yule_amd.backend import NO_TOKEN, YuleGpuError

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dt,heads,kv,hd,lens,slots,split", batch_shapes.PROMPTS)
@pytest.mark.parametrize("bad", [None, NAN, INF])
def test_prompt_attn_split(hip, dt, heads, kv, hd, lens, slots, split, bad):
    """bad: in rows of K and V that the checked rows do not see."""
    say(f"[batch] prompt_attn {dt.name} {heads}/{kv}x{hd} lens {lens}, hidden {bad}")
    n = sum(lens)
    q, k, v = normal(1, (n, heads * hd), dt, 1.5), normal(2, (n, kv * hd), dt), normal(3, (n, kv * hd), dt)
    rows = [0, 1, 31, 32, 63, 64, 65, 127, 128, 129, 500, 767, 768]
    if bad is None:
        rows += [n - 66, n - 2, n - 1]
    want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt, set(rows))
    if bad is not None:
        v[769], k[771] = bad, bad
    with Dev(hip) as d:
        out = d.new(q.numel() * 2)
        hip.prompt_attn(d.up(q), d.up(k), d.up(v), out, d.up(np.cumsum([0] + lens).astype(np.uint32)), len(lens), n, heads, kv, hd, dt)
        got = d.down(out, tuple(q.shape), dt)
    check(got[rows], want[rows], bound[rows], "prompt_attn")
    if bad is not None:
        seen = got[769:771].float()
        assert (seen == bad).all() if bad == bad else torch.isnan(seen).all()


@pytest.mark.parametrize("dt", list(TYPES), ids=lambda d: d.name)
@pytest.mark.parametrize("shape", [s for s, *_ in batch_shapes.PREFIXES] + batch_shapes.SHORT, ids=lambda s: "x".join(str(s[i]) for i in (0, 1, 2, 3)))
@pytest.mark.parametrize("bad", [None, NAN, INF])
def test_prefix_attn_chunks(hip, dt, shape, bad):
    """bad: one value of V in the prefix' last row, in a tile that the prefix does not fill, which every row sees, and V's rows
    behind the tails."""
    heads, kv, hd, prefix, cap, lens, tokens = shape
    say(f"[batch] prefix_attn {dt.name} {heads}/{kv}x{hd} prefix {prefix}, {len(lens)} tails of {cap}, {tokens} tokens, {bad}")
    q, kp, vp, kt, vt = prefix_inputs(20, heads, kv, hd, prefix, cap, lens, tokens, dt)
    dim = kv * hd - 1   # of the last KV head
    if bad is not None:
        vp[prefix - 1, dim] = 0
    seqs = [0, len(lens) // 2, len(lens) - 1]
    parts = [prefix_reference(q[s * tokens:(s + 1) * tokens], kp, vp, kt[s * cap:(s + 1) * cap], vt[s * cap:(s + 1) * cap],
                              [lens[s]], cap, tokens, heads, kv, hd, dt) for s in seqs]
    want, bound = (torch.cat([p[i] for p in parts]) for i in (0, 1))
    if bad is not None:
        vp[prefix - 1, dim] = bad
        for s, n in enumerate(lens):
            vt[s * cap + n:(s + 1) * cap] = bad
    with Dev(hip) as d:
        got = run_prefix(hip, d, q, kp, vp, kt, vt, lens, cap, tokens, heads, kv, hd, dt)
    got = torch.cat([got[s * tokens:(s + 1) * tokens] for s in seqs])
    has = torch.zeros(got.shape, dtype=torch.bool)
    if bad is not None:
        has[:, heads * hd - heads // kv * hd + hd - 1::hd] = True
        seen = got[has].float()
        assert (seen == bad).all() if bad == bad else torch.isnan(seen).all()
    check(got[~has], want[~has], bound[~has], "prefix_attn")


# ---------------------------------------------------------------- verification: weights that are multiples of 2^-20, whose sums
# are exact in any order
def dyadic(rng, *shape):
    return (rng.integers(0, 1 << 10, shape) / (1 << 20)).astype(np.float32)


@pytest.mark.parametrize("vocab", [4097, 9000, 300001])
@pytest.mark.parametrize("u_last", [0.0, 0.3, float(np.float32(1 - 2.0 ** -24)), 1.0])
def test_verify_drafts_many_chunks(hip, vocab, u_last):
    """Rows of several chunks, and of more than 64: a draft that is not kept where p = q everywhere (the token is of p then),
    a draft that is no token, all kept, weights in the last chunk alone or in the first alone, none at all."""
    say(f"[batch] verify_drafts, {vocab} values, u {u_last}")
    rng = np.random.default_rng(vocab)
    b, n = 9, 2
    p, q = dyadic(rng, b, n + 1, vocab), dyadic(rng, b, n, vocab)
    drafts, u = rng.integers(0, vocab, (b, n)).astype(np.uint32), np.full((b, n + 1), u_last, np.float32)
    u[:, :n] = 0.999
    q[0] = p[0, :n]                                   # p = q: not kept where it is 0
    p[0, 0, drafts[0, 0]] = q[0, 0, drafts[0, 0]] = 0
    q[1] = p[1, :n]                                   # p = q, and the draft is no token
    drafts[1, 0] = vocab + 5
    q[2] = p[2, :n] / 2                               # all kept where p > 0
    p[2, [0, 1], drafts[2]] = 0.25
    p[3, :, :vocab - 3] = 0                           # weights at the end only
    q[3] = 0
    p[3, :2, drafts[3]] = 0
    p[4, :, 40:], q[4] = 0, 0                         # at the beginning only: chunks behind without any
    p[5], q[5] = 0, .5                                # none
    p[6], q[6] = NAN, .5
    p[7] = -1
    p[7, 0, vocab - 1], q[7, 0] = .5, p[7, 0]         # p = q, negative but for the last value
    drafts[7, 0] = 0
    with Dev(hip) as d:
        first = run_verify(hip, d, p, q, drafts, u, None, vocab)
        again = run_verify(hip, d, p, q, drafts, u, None, vocab)
    wa, wt = verify_reference(p, q, drafts, u, [n] * b, vocab)
    for acc, tok in (first, again):
        assert np.array_equal(acc, wa) and np.array_equal(tok, wt)
    assert wa[0] == wa[1] == 0 and wa[2] == 2 and wt[5, 0] == wt[6, 0] == NO_TOKEN and wt[7, 0] == vocab - 1


@pytest.mark.parametrize("at", [0, 4095, 4096, 64 * 4096 - 1, 64 * 4096, 299999])
def test_verify_drafts_one_weight(hip, at):
    """Plain sampling of a row with one weight, wherever it is."""
    say(f"[batch] verify_drafts, one weight at {at}")
    vocab = 300000
    p = np.zeros((3, 1, vocab), np.float32)
    p[:, 0, at] = [1, 1e-30, 3]
    u = np.array([[0], [.5], [1 - 2.0 ** -24]], np.float32)
    with Dev(hip) as d:
        acc, tok = run_verify(hip, d, p, p[:, :0], np.zeros((3, 0), np.uint32), u, None, vocab)
    assert (acc == 0).all() and (tok == at).all()


def test_verify_drafts_many_sequences(hip):
    """More sequences than one launch takes, with tickets: the second launch uses the first one's."""
    b, n, vocab = 1100, 1, 4097
    say(f"[batch] verify_drafts, {b} sequences of {vocab}")
    rng = np.random.default_rng(7)
    p, q = dyadic(rng, b, n + 1, vocab), dyadic(rng, b, n, vocab)
    drafts, u = rng.integers(0, vocab, (b, n)).astype(np.uint32), rng.random((b, n + 1), np.float32)
    with Dev(hip) as d:
        got = [run_verify(hip, d, p, q, drafts, u, None, vocab) for _ in range(2)]
    wa, wt = verify_reference(p, q, drafts, u, [n] * b, vocab)
    for acc, tok in got:
        assert np.array_equal(acc, wa) and np.array_equal(tok, wt)


def test_verify_drafts_wide_vocabulary(hip):
    """Rows of 2^24 values and more."""
    vocab = (1 << 24) + 5
    say(f"[batch] verify_drafts, {vocab} values")
    p, q = torch.zeros(4, vocab, device="cuda"), torch.zeros(2, vocab, device="cuda")
    x = 1 << 24
    p[0, 3], p[0, x + 4], p[0, x + 1], q[0, x + 1] = .25, .5, .25, .5   # draft x + 1: .75 * .5 >= .25, weights .25 and .5
    p[2, x + 2], q[1, x + 2] = .5, .5                                   # kept
    p[3, 64 * 4096 + 7], p[3, x] = .5, .5                               # the sum has to pass .5
    p[1], p[3, 5] = float("nan"), -1                                    # (not looked at; no weight)
    ids = torch.tensor([x + 1, x + 2], dtype=torch.int32, device="cuda")
    u = torch.tensor([[.75, .5], [.75, .5]], device="cuda")
    acc, tok = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (2, 4))
    torch.cuda.synchronize()
    h = [hip.import_buffer(t.data_ptr(), t.numel() * 4) for t in (p, q, ids, u, acc, tok)]
    hip.verify_drafts(h[0], h[1], h[2], h[3], None, h[4], h[5], 2, 1, vocab)
    hip.synchronize()
    assert acc.tolist() == [0, 1] and tok.tolist() == [x + 4, -1, x + 2, x]
    for b in h:
        hip.free(b)


def test_limits(hip):
    """The most rows that a call takes, and one more."""
    say("[batch] limits of a launch")
    most, tokens = 1 << 23, 64
    q, k, v = (torch.ones(n, 8, dtype=torch.float16, device="cuda") for n in (most + tokens, 1, 1))
    v[0] = torch.arange(8)
    out, ints = torch.zeros_like(q), torch.zeros(most + 8, dtype=torch.int32, device="cuda")
    p, other = torch.ones(most + 8, device="cuda"), torch.zeros(most + 8, dtype=torch.int32, device="cuda")
    small = torch.zeros(16, 8, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    hq, hk, hv, ho, hi, hp, hx, hs = h = [hip.import_buffer(t.data_ptr(), t.numel() * t.element_size())
                                          for t in (q, k, v, out, ints, p, other, small)]
    u = hip.upload(np.full(most + 8, .5, np.float32))
    for n, call in ((most // tokens, lambda n: hip.prefix_attn(hq, hk, hv, 1, None, None, hi, 0, ho, n, tokens, 1, 1, 8, 1)),
                    (most, lambda n: hip.verify_drafts(hp, None, None, u, None, hi, hx, n, 0, 1)),
                    (most, lambda n: hip.prompt_attn(hq, hq, hq, hs, hi, n, 10, 1, 1, 8, 1))):
        with pytest.raises(YuleGpuError) as e:
            call(n + 1)
        assert e.value.code == 1 and "too many rows" in str(e.value)
        if n < most:
            call(n)
            hip.synchronize()
            assert bool((out[:most] == v[0]).all()) and not bool(out[most:].any())
    for x in (*h, u):
        hip.free(x)
