"""The operators of a batched, speculative serving step, as cases to be timed and compared.

  prompt   causal attention with grouped heads over packed prompts of different lengths (prompt_attn)
  prefix   attention of each sequence's newest tokens over a prefix that the whole batch shares and the
           sequence's own tail (prefix_attn)
  verify   acceptance of drafted tokens against the target's probabilities from given random numbers, and the
           token that follows them (verify_drafts; without drafts it is plain sampling)

`own` false: elementary torch operations in 32 bits (64 for the cumulative sums of a vocabulary); true: the calls
of `yule_amd.backend.HipBackend`.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_TYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
_NO_TOKEN = 0xFFFFFFFF


def listed():
    return [
        # three chat turns of a few tokens arriving together: launch latency
        {"name": "prompt_small", "kind": "prompt", "dtype": "F32", "heads": 32, "kv_heads": 4, "head_dim": 64,
         "lens": "5 1 11", "spare": 0, "fused": False},
        # an admission batch of ragged prompts, q, k and v as slices of one projection's rows, the buffer longer
        # than the batch
        {"name": "prompt_ragged", "kind": "prompt", "dtype": "F16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "lens": "333 1 128 777 64 0 511", "spare": 234, "fused": True},
        # the f32 path of the framework's own model: a long and an ordinary prompt
        {"name": "prompt_f32", "kind": "prompt", "dtype": "F32", "heads": 32, "kv_heads": 4, "head_dim": 64,
         "lens": "1531 128", "spare": 0, "fused": False},
        # documents to be summarised: matrix-core rate
        {"name": "prompt_long", "kind": "prompt", "dtype": "BF16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "lens": "4096 2777 4001", "spare": 0, "fused": False},
        # two requests behind a short system prompt: launch latency
        {"name": "prefix_small", "kind": "prefix", "dtype": "F32", "heads": 32, "kv_heads": 4, "head_dim": 64,
         "seqs": 2, "tokens": 1, "prefix": 128, "tail": 64},
        # eight requests, four drafts and the last token of each scored together
        {"name": "prefix_drafts", "kind": "prefix", "dtype": "BF16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "seqs": 8, "tokens": 5, "prefix": 2048, "tail": 777},
        # a long shared document, heads of 80 dims, odd batch and lengths
        {"name": "prefix_odd", "kind": "prefix", "dtype": "F16", "heads": 12, "kv_heads": 2, "head_dim": 80,
         "seqs": 13, "tokens": 1, "prefix": 15001, "tail": 100},
        # an f32 cache at the 8B width
        {"name": "prefix_f32", "kind": "prefix", "dtype": "F32", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "seqs": 16, "tokens": 1, "prefix": 8192, "tail": 300},
        # a full batch over a long shared document, each with an answer under way
        {"name": "prefix_long", "kind": "prefix", "dtype": "BF16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "seqs": 64, "tokens": 1, "prefix": 32768, "tail": 1024},
        # one user's request: latency
        {"name": "verify_one", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "ragged": False},
        # a batch of them, with fewer drafts where a request nears its limit
        {"name": "verify_batch", "kind": "verify", "seqs": 64, "drafts": 5, "vocab": 32000, "ragged": True},
        # the widest vocabulary
        {"name": "verify_wide", "kind": "verify", "seqs": 16, "drafts": 7, "vocab": 128256, "ragged": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("prompt", "prefix", "verify"))
    if kind == "verify":
        vocab = _log_int(rng, 1000, 128256)
        return {"kind": kind, "seqs": _log_int(rng, 1, min(64, 2050000 // vocab)), "drafts": rng.randint(0, 12),
                "vocab": vocab, "ragged": rng.choice((False, True))}
    heads, kv_heads = rng.choice(((32, 4), (32, 8), (12, 2), (16, 16)))
    case = {"kind": kind, "dtype": rng.choice(tuple(_TYPES)), "heads": heads, "kv_heads": kv_heads,
            "head_dim": rng.choice((64, 80, 128))}
    if kind == "prompt":
        # f32 products run at a fraction of the 16-bit rate
        most = 1600 if case["dtype"] == "F32" else 4096
        lens = [_log_int(rng, 1, most) for _ in range(rng.choice((1, 2, 3, 3, 9)))]
        if len(lens) > 3:
            lens = [1 + n // 3 for n in lens]
        return {**case, "lens": " ".join(map(str, lens)), "spare": rng.choice((0, 0, 77)),
                "fused": rng.choice((False, True))}
    seqs, tokens = _log_int(rng, 1, 64), rng.choice((1, 1, 2, 5, 8))
    # rows of a cache of 64 MiB for K and as much for V
    rows = (64 << 20) // (kv_heads * case["head_dim"] * (4 if case["dtype"] == "F32" else 2))
    return {**case, "seqs": seqs, "tokens": tokens, "prefix": _log_int(rng, 16, min(16000, rows)),
            "tail": tokens + _log_int(rng, 1, min(700, rows // seqs - 8))}


# ---------------------------------------------------------------- inputs
def _lens(case):
    return [int(n) for n in case["lens"].split()]


def _tail_lens(case):
    """Rows of each sequence's tail, its newest tokens among them: spread over what its cache can hold."""
    n = case["tokens"]
    return [n + 7919 * (s + 1) % (case["tail"] - n + 1) for s in range(case["seqs"])]


def _draft_lens(case):
    return [case["drafts"] - (s % 3 if case["ragged"] else 0) if case["drafts"] >= 3 else case["drafts"]
            for s in range(case["seqs"])]


def _inputs(case, seed):
    """A case's tensors, from its seed alone."""
    g = torch.Generator(device=_DEV).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=None):
        t = torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32) * scale
        return t.to(dtype) if dtype is not None else t

    if case["kind"] == "verify":
        b, n, vocab = case["seqs"], case["drafts"], case["vocab"]
        logits = normal(b, n + 1, vocab, scale=3.0)
        # a drafting model is nearly right: its logits are the target's with an error
        p = torch.softmax(logits, -1)
        q = torch.softmax(logits[:, :n] + normal(b, n, vocab, scale=0.7), -1)
        # drafts are drawn from the drafting model's probabilities (the largest of p / exponential variates)
        e = torch.rand((b, n, vocab), generator=g, device=_DEV).clamp_min(1e-12).log().neg()
        drafts = (q / e).argmax(-1).to(torch.int32) if n else torch.zeros((b, 0), dtype=torch.int32, device=_DEV)
        return {"p": p, "q": q, "drafts": drafts, "uniforms": torch.rand((b, n + 1), generator=g, device=_DEV),
                "lens": torch.tensor(_draft_lens(case), dtype=torch.int32, device=_DEV)}
    dt, hd = _TYPES[case["dtype"]], case["head_dim"]
    qd, kvd = case["heads"] * hd, case["kv_heads"] * hd
    # queries of norm well above one, so that some heads attend to few keys and others to many
    if case["kind"] == "prompt":
        rows = sum(_lens(case)) + case["spare"]
        got = {"q": normal(rows, qd, scale=1.5, dtype=dt), "k": normal(rows, kvd, dtype=dt),
               "v": normal(rows, kvd, dtype=dt)}
        if case["fused"]:
            got = {"qkv": torch.cat([got["q"], got["k"], got["v"]], 1)}
        # what the rows behind the last sequence hold stays there
        return {**got, "out": torch.full((rows, qd), 0.5, dtype=dt, device=_DEV),
                "offsets": torch.tensor([0] + list(np.cumsum(_lens(case))), dtype=torch.int32, device=_DEV)}
    b, n = case["seqs"], case["tokens"]
    return {"q": normal(b * n, qd, scale=1.5, dtype=dt),
            "k_prefix": normal(case["prefix"], kvd, dtype=dt), "v_prefix": normal(case["prefix"], kvd, dtype=dt),
            "k_tail": normal(b * case["tail"], kvd, dtype=dt), "v_tail": normal(b * case["tail"], kvd, dtype=dt),
            "tail_lens": torch.tensor(_tail_lens(case), dtype=torch.int32, device=_DEV)}


# ---------------------------------------------------------------- the framework's side
_backend = None


def _hip():
    """The program's backend: one per process, as its stream and buffers are."""
    global _backend
    if _backend is None:
        from yule_amd.backend import HipBackend
        _backend = HipBackend(0)
    return _backend


class Handles:
    """The backend's handles over a case's tensors, by name: the tensors are read and written where they lie."""

    def __init__(self, hip, tensors):
        self.hip, self.tensors = hip, tensors
        self.h = {name: hip.import_buffer(t.data_ptr(), t.numel() * t.element_size()) if t.numel() else None
                  for name, t in tensors.items()}

    def __del__(self):
        for h in getattr(self, "h", {}).values():
            if h is not None:
                self.hip.free(h)


class State:
    def __init__(self, case, tensors):
        self.case = case
        self.t = tensors


def prepare(case, seed):
    st = State(case, _inputs(case, seed))
    if own:
        from yule_amd import DType
        from yule_amd.backend import Rows
        hip, kind, n_seqs = _hip(), case["kind"], case.get("seqs")
        # the program's stream is the backend's: torch's work and the operators' follow each other on it
        stream = torch.cuda.ExternalStream(hip.stream)
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        if kind == "verify":
            # the ids that the operator writes, 32 bits each, and the program's 64-bit tokens
            at, shape = -(-n_seqs // 4) * 4, (n_seqs, case["drafts"] + 1)
            ids = torch.zeros(at + shape[0] * shape[1], dtype=torch.int32, device=_DEV)
            st.t["accepted"], st.t["tokens"] = ids[:n_seqs], ids[at:]
            st.ids, st.wide = ids.view(torch.uint32), torch.zeros(ids.shape, dtype=torch.int64, device=_DEV)
            st.result = {"accepted": st.wide[:n_seqs], "tokens": st.wide[at:].view(shape)}
        else:
            if kind == "prefix":
                st.t["out"] = torch.zeros_like(st.t["q"])
            else:
                st.n_seqs, st.n_rows = st.t["offsets"].numel() - 1, st.t["out"].shape[0]
            st.result = {"out": st.t["out"]}
            st.dtype = DType[case["dtype"]]
        st.b = Handles(hip, st.t)
        h = st.b.h
        if kind == "verify":
            st.rows = {n: Rows(h[n], case["vocab"]) if h[n] is not None else None for n in ("p", "q")}
        else:
            qd, kvd = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
            if kind == "prompt" and case["fused"]:
                ld = qd + 2 * kvd
                st.rows = {"q": Rows(h["qkv"], ld), "k": Rows(h["qkv"], ld, qd), "v": Rows(h["qkv"], ld, qd + kvd)}
            else:
                st.rows = {n: Rows(h[n], qd if n == "q" else kvd) for n in h if n.split("_")[0] in ("q", "k", "v")}
            st.rows["out"] = Rows(h["out"], qd)
    return st


def _run_own(st):
    hip, case, h, rows = st.b.hip, st.case, st.b.h, st.rows
    if case["kind"] == "prompt":
        hip.prompt_attn(rows["q"], rows["k"], rows["v"], rows["out"], h["offsets"], st.n_seqs, st.n_rows,
                        case["heads"], case["kv_heads"], case["head_dim"], st.dtype)
    elif case["kind"] == "prefix":
        hip.prefix_attn(rows["q"], rows["k_prefix"], rows["v_prefix"], case["prefix"], rows["k_tail"], rows["v_tail"],
                        h["tail_lens"], case["tail"], rows["out"], case["seqs"], case["tokens"], case["heads"],
                        case["kv_heads"], case["head_dim"], st.dtype)
    else:
        hip.verify_drafts(rows["p"], rows["q"], h["drafts"], h["uniforms"], h["lens"], h["accepted"], h["tokens"],
                          case["seqs"], case["drafts"], case["vocab"])
        st.wide.copy_(st.ids)
    return st.result


# ---------------------------------------------------------------- the plain forms
def _weights(scores, hidden):
    """Softmax over the last axis of masked scores; rows that see nothing get zeros."""
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_prompt(st):
    case, t = st.case, st.t
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lens = _lens(case)
    longest, n, total, group = max(lens), len(lens), sum(lens), heads // kv
    q, k, v = t["qkv"].split([heads * hd, kv * hd, kv * hd], 1) if case["fused"] else (t["q"], t["k"], t["v"])
    at = torch.arange(longest, device=_DEV)
    off = t["offsets"].long()
    valid = at[None, :] < (off[1:] - off[:-1])[:, None]                       # [n, longest]
    rows = torch.where(valid, off[:-1, None] + at[None, :], 0)
    q = q[rows].float().view(n, longest, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, group * longest, hd)
    k = k[rows].float().view(n, longest, kv, hd).permute(0, 2, 3, 1).contiguous()
    v = v[rows].float().view(n, longest, kv, hd).permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).view(n, kv, group, longest, longest)
    hidden = (at[None, :] > at[:, None]) | ~valid[:, None, None, None, :]
    out = torch.matmul(_weights(scores, hidden).view(n, kv, group * longest, longest), v)
    out = out.view(n, kv, group, longest, hd).permute(0, 3, 1, 2, 4).reshape(n, longest, heads * hd)
    t["out"][:total] = out[valid].to(t["out"].dtype)
    return {"out": t["out"]}


def _plain_prefix(st):
    case, t = st.case, st.t
    kv, hd, b, n, cap, p = case["kv_heads"], case["head_dim"], case["seqs"], case["tokens"], case["tail"], case["prefix"]
    group = case["heads"] // kv
    q = t["q"].float().view(b, n, kv, group, hd).permute(2, 0, 1, 3, 4)       # [kv, b, n, group, hd]
    kp = t["k_prefix"].float().view(p, kv, hd).permute(1, 2, 0).contiguous()
    vp = t["v_prefix"].float().view(p, kv, hd).permute(1, 0, 2).contiguous()
    kt = t["k_tail"].float().view(b, cap, kv, hd).permute(2, 0, 3, 1).contiguous()
    vt = t["v_tail"].float().view(b, cap, kv, hd).permute(2, 0, 1, 3).contiguous()
    s1 = torch.matmul(q.reshape(kv, b * n * group, hd), kp).view(kv, b, n, group, p)
    s2 = torch.matmul(q.reshape(kv, b, n * group, hd), kt).view(kv, b, n, group, cap)
    last = t["tail_lens"].long()[:, None] - n + torch.arange(n, device=_DEV)[None, :]   # newest visible row
    hidden = torch.arange(cap, device=_DEV)[None, None, :] > last[:, :, None]           # [b, n, cap]
    hidden = torch.cat([hidden.new_zeros(b, n, p), hidden], -1)[None, :, :, None, :]
    w = _weights(torch.cat([s1, s2], -1) / math.sqrt(hd), hidden)
    out = torch.matmul(w[..., :p].reshape(kv, b * n * group, p), vp).view(kv, b, n, group, hd)
    out += torch.matmul(w[..., p:].reshape(kv, b, n * group, cap), vt).view(kv, b, n, group, hd)
    return {"out": out.permute(1, 2, 0, 3, 4).reshape(b * n, kv * group * hd).to(t["q"].dtype)}


def _plain_verify(st):
    case, t = st.case, st.t
    b, n, vocab = case["seqs"], case["drafts"], case["vocab"]
    lens, x, u = t["lens"].long(), t["drafts"].long(), t["uniforms"].double()
    at = torch.arange(n, device=_DEV)
    px = torch.gather(t["p"][:, :n], 2, x[:, :, None])[:, :, 0].double()
    qx = torch.gather(t["q"], 2, x[:, :, None])[:, :, 0].double()
    stop = ~(u[:, :n] * qx < px) | (at[None, :] >= lens[:, None])
    accepted = torch.cumprod((~stop).long(), 1).sum(1)
    seq = torch.arange(b, device=_DEV)
    p = t["p"][seq, accepted].double()
    if n:
        q = t["q"][seq, accepted.clamp_max(n - 1)].double()
        rest = (p - q).clamp_min(0.0)
        rejected = (accepted < lens) & (rest.amax(1) > 0)
        p = torch.where(rejected[:, None], rest, p)
    c = torch.cumsum(p, 1)
    below = (c <= (u[:, n] * c[:, -1])[:, None]).sum(1)
    some = torch.where(p > 0, torch.arange(vocab, device=_DEV)[None, :], -1).amax(1)
    nxt = torch.minimum(below, some)
    col = torch.arange(n + 1, device=_DEV)[None, :]
    drafts = torch.cat([x, x.new_zeros(b, 1)], 1)
    tokens = torch.where(col < accepted[:, None], drafts,
                         torch.where(col == accepted[:, None], nxt[:, None], _NO_TOKEN))
    return {"accepted": accepted, "tokens": tokens}


def run(st):
    if own:
        return _run_own(st)
    return {"prompt": _plain_prompt, "prefix": _plain_prefix, "verify": _plain_verify}[st.case["kind"]](st)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "verify":
        b, n, vocab = case["seqs"], case["drafts"], case["vocab"]
        # one row of each distribution (the target's alone without drafts), the drafts' own probabilities, the answer
        return {"bytes": b * (vocab * (8 if n else 4) + 20 * n + 8 * (n + 2)), "flops": 3 * b * vocab}
    size = torch.empty((), dtype=_TYPES[case["dtype"]]).element_size()
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "prompt":
        total, pairs = sum(_lens(case)), sum(n * (n + 1) // 2 for n in _lens(case))
        return {"bytes": 2 * total * (heads + kv) * hd * size + 4 * (len(_lens(case)) + 1), "flops": 4 * hd * heads * pairs}
    n, tails = case["tokens"], _tail_lens(case)
    queries, keys = case["seqs"] * n, case["prefix"] + sum(tails)
    pairs = queries * case["prefix"] + sum(n * m - n * (n - 1) // 2 for m in tails)
    return {"bytes": 2 * (queries * heads + keys * kv) * hd * size + 4 * case["seqs"], "flops": 4 * hd * heads * pairs}


# ---------------------------------------------------------------- the same in 64 bits
def _attend64(q, k, v, seen):
    """One head's [rows, hd] results: row r sees the first seen[r] keys (f64, a slab of rows at a time)."""
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    if not k.shape[0]:
        return out
    scale, key = 1.0 / math.sqrt(q.shape[1]), torch.arange(k.shape[0], device=q.device)
    kt = k.T.contiguous()
    for r0 in range(0, q.shape[0], 2048):
        s = (q[r0:r0 + 2048] @ kt) * scale
        gone = key[None, :] >= seen[r0:r0 + 2048, None]
        s[gone] = -math.inf
        some = (seen[r0:r0 + 2048] > 0)[:, None]
        w = torch.softmax(torch.where(some, s, 0.0), 1)
        out[r0:r0 + 2048] = torch.where(some, w @ v, 0.0)
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(case, {k: v.cpu().numpy() for k, v in t.items()})
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    group = heads // kv
    if case["kind"] == "prompt":
        if case["fused"]:
            t["q"], t["k"], t["v"] = (x.contiguous() for x in t["qkv"].split([heads * hd, kv * hd, kv * hd], 1))
        q, k, v, out = (t[n].double() for n in ("q", "k", "v", "out"))
        at = 0
        for m in _lens(case):
            seen = torch.arange(1, m + 1, device=_DEV)
            for h in range(heads):
                qc, kc = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
                out[at:at + m, qc] = _attend64(q[at:at + m, qc], k[at:at + m, kc], v[at:at + m, kc], seen)
            at += m
        return {"out": out}
    n, cap = case["tokens"], case["tail"]
    t = {k: v.double() if v.is_floating_point() else v for k, v in t.items()}
    out = torch.empty_like(t["q"])
    for s, m in enumerate(_tail_lens(case)):
        r = slice(s * n, (s + 1) * n)
        for g in range(kv):
            c = slice(g * hd, (g + 1) * hd)
            k = torch.cat([t["k_prefix"][:, c], t["k_tail"][s * cap:s * cap + m, c]])
            v = torch.cat([t["v_prefix"][:, c], t["v_tail"][s * cap:s * cap + m, c]])
            q = t["q"][r, g * group * hd:(g + 1) * group * hd].reshape(n * group, hd)
            seen = (case["prefix"] + m - n + 1 + torch.arange(n, device=_DEV)).repeat_interleave(group)
            out[r, g * group * hd:(g + 1) * group * hd] = _attend64(q, k, v, seen).view(n, group * hd)
    return {"out": out}


def _exact_verify(case, t):
    b, n = case["seqs"], case["drafts"]
    accepted, tokens = np.zeros(b, np.int64), np.full((b, n + 1), _NO_TOKEN, np.int64)
    for s in range(b):
        a = 0
        while a < t["lens"][s]:
            x = t["drafts"][s, a]
            if not float(t["uniforms"][s, a]) * float(t["q"][s, a, x]) < float(t["p"][s, a, x]):
                break
            tokens[s, a] = x
            a += 1
        w = t["p"][s, a].astype(np.float64)
        if a < t["lens"][s]:
            rest = np.maximum(w - t["q"][s, a].astype(np.float64), 0.0)
            w = rest if rest.any() else w
        c = np.cumsum(w)
        past = np.nonzero(c > float(t["uniforms"][s, n]) * c[-1])[0]
        accepted[s], tokens[s, a] = a, past[0] if past.size else np.nonzero(w)[0][-1]
    return {"accepted": accepted, "tokens": tokens}
