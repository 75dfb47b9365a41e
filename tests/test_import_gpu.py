"""Device memory of the caller's under the backend's handles: tensors of torch's
as arguments where they lie, on the backend's stream; what is refused; whose the
memory stays."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_batch_gpu import (Dev, bits_of, check, normal, prefix_inputs, prefix_reference, prompt_reference, run_verify, say,
                            verify_inputs)
from yule_amd import DType, synth
from yule_amd.backend import HipBackend, Rows, YuleGpuError

pytestmark = pytest.mark.gpu


@pytest.fixture
def torch_on(hip):
    """torch's work goes to the backend's stream."""
    with torch.cuda.stream(torch.cuda.ExternalStream(hip.stream)):
        yield


class Imported:
    """Handles over tensors, freed at the end."""

    def __init__(self, hip):
        self.hip, self.h, self.kept = hip, [], []

    def __call__(self, t):
        assert t.is_contiguous()
        self.kept.append(t)
        self.h.append(self.hip.import_buffer(t.data_ptr(), t.numel() * t.element_size()))
        return self.h[-1]

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for h in self.h:
            self.hip.free(h)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_operators_on_tensors(hip, torch_on):
    """A fused projection by torch, attention where its rows lie, torch on the results: no synchronization in between, and
    the same results as from uploaded copies."""
    say("[import] prompt_attn, prefix_attn and verify_drafts on torch's tensors")
    heads, kv, hd, lens, dt = 8, 2, 64, [70, 3, 41], DType.BF16
    n, ld = sum(lens), (heads + 2 * kv) * hd
    x, w = normal(1, (n, 256), dt).cuda(), normal(2, (256, ld), dt, 256 ** -.5).cuda()
    qkv, out = torch.empty(n, ld, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, heads * hd, dtype=torch.bfloat16, device="cuda")
    offs = ints(np.cumsum([0] + lens).tolist())
    with Imported(hip) as imp:
        h, ho, hoff = imp(qkv), imp(out), imp(offs)
        for scale in (1.0, 1.5):   # the handles stay, the contents change
            torch.mm(x * scale, w, out=qkv)
            hip.prompt_attn(Rows(h, ld), Rows(h, ld, heads * hd), Rows(h, ld, (heads + kv) * hd), ho, hoff, len(lens), n, heads,
                            kv, hd, dt)
            got, doubled = out.clone(), out * 2
            assert torch.equal(doubled, got * 2)
            q, k, v = qkv.cpu().split([heads * hd, kv * hd, kv * hd], 1)
            want, bound = prompt_reference(q, k, v, lens, heads, kv, hd, dt)
            check(got.cpu(), want, bound, "prompt_attn")
    prefix, cap, tails, tokens = 600, 30, [30, 4, 11], 2
    t = prefix_inputs(5, heads, kv, hd, prefix, cap, tails, tokens, dt)
    dev = [x.cuda() for x in t]
    out = torch.empty_like(dev[0])
    with Imported(hip) as imp:
        q, kp, vp, kt, vt = (imp(x) for x in dev)
        hip.prefix_attn(q, kp, vp, prefix, kt, vt, imp(ints(tails)), cap, imp(out), len(tails), tokens, heads, kv, hd, dt)
        got = out.cpu()
    want, bound = prefix_reference(*t, tails, cap, tokens, heads, kv, hd, dt)
    check(got, want, bound, "prefix_attn")
    b, n, vocab = 5, 3, 5000
    p, pq, drafts, u = verify_inputs(6, b, n, vocab)
    acc, tok = ints([0] * b), ints([[0] * (n + 1)] * b)
    with Imported(hip) as imp:
        hip.verify_drafts(imp(torch.from_numpy(p).cuda()), imp(torch.from_numpy(pq).cuda()), imp(ints(drafts.tolist())),
                          imp(torch.from_numpy(u).cuda()), None, imp(acc), imp(tok), b, n, vocab)
        got = acc.cpu().numpy().view(np.uint32), tok.cpu().numpy().view(np.uint32)
    with Dev(hip) as d:
        want = run_verify(hip, d, p, pq, drafts, u, None, vocab)
    assert all(np.array_equal(g, w) for g, w in zip(got, want))


def test_captured_with_tensors(hip):
    """Calls on imported memory in a captured graph, replayed after torch has changed the memory."""
    say("[import] capture and replay")
    be = HipBackend(0)
    heads, kv, hd, n, dt = 4, 2, 64, 50, DType.F32
    with torch.cuda.stream(torch.cuda.ExternalStream(be.stream)):
        x = [normal(7 + i, (n, w * hd), dt).cuda() for i, w in enumerate((heads, kv, kv))]
        out, offs = torch.empty_like(x[0]), ints([0, n])
        with Imported(be) as imp:
            args = (*(imp(t) for t in x), imp(out), imp(offs), 1, n, heads, kv, hd, dt)
            be.prompt_attn(*args)
            be.capture_begin()
            be.prompt_attn(*args)
            be.capture_end()
            for i in range(3):
                x[0].mul_(0.5 + i)
                x[2].add_(1)
                out.zero_()
                be.capture_replay()
                got = out.clone()
                be.prompt_attn(*args)
                assert torch.equal(bits_of(got), bits_of(out)) and bool(got.any())
        torch.cuda.current_stream().synchronize()
    be.close()


def test_memory_stays_the_callers(hip, torch_on):
    say("[import] free and close leave the memory alone")
    t = torch.arange(1000, dtype=torch.float32, device="cuda")
    h = hip.import_buffer(t.data_ptr(), 4000)
    assert np.array_equal(hip.download(h, 1000), np.arange(1000, dtype=np.float32))
    hip.copy_to_device(np.full(1000, 3, np.float32), h)
    assert bool((t == 3).all())
    own = hip.upload(np.full(1000, 5, np.float32))
    hip.copy_buffer(own, h, 4000)
    assert bool((t == 5).all())
    hip.free(h)
    hip.free(own)
    with pytest.raises(YuleGpuError) as e:
        hip.download(h, 1)
    assert e.value.code == 1
    be = HipBackend(0)
    h = be.import_buffer(t.data_ptr(), 4000)   # (a handle is of one backend)
    be.close()
    assert bool((t == 5).all())
    t.add_(1)
    assert bool((t == 6).all())


def test_refusals(hip, torch_on):
    say("[import] refusals")
    t, host = torch.zeros(4096, dtype=torch.float32, device="cuda"), np.zeros(1024, np.float32)
    a, pinned = t.data_ptr(), torch.zeros(1024, pin_memory=True)
    big = torch.cuda.get_device_properties(0).total_memory
    for ptr, size in [(None, 16), (a, 0), (a + 8, 16), (host.ctypes.data // 16 * 16 + 16, 64), (pinned.data_ptr(), 64), (a, big),
                      (a, 2 ** 64 - 16), (a, 2 ** 64 - 1)]:
        with pytest.raises(YuleGpuError) as e:
            hip.import_buffer(ptr, size)
        assert e.value.code == 1, (ptr, size)
    assert hip._lib.yule_hip_import_buffer(hip.raw, a, 16, None) == 1 and hip._lib.yule_hip_stream(hip.raw, None) == 1
    h = hip.import_buffer(a + 1024, 1024)
    for ptr, size in [(a, 16384), (a + 1024, 1024), (a + 1024, 16), (a + 2032, 64), (a + 1008, 32)]:
        with pytest.raises(YuleGpuError) as e:
            hip.import_buffer(ptr, size)
        assert e.value.code == 1 and "overlaps" in str(e.value)
    others = [hip.import_buffer(a, 1024), hip.import_buffer(a + 2048, 16)]
    for x in (h, *others):
        hip.free(x)
    h = hip.import_buffer(a, 16384)   # free again
    with pytest.raises(YuleGpuError):
        hip.copy_to_device(np.zeros(4097, np.float32), h)
    hip.free(h)
    hip.synchronize()


def test_other_calls_keep_their_slack(hip, torch_on):
    """Entries whose kernels may read past their data take imported memory that has 64 bytes more."""
    say("[import] quantized_matmul on imported weights")
    rows, cols = 64, 256
    w = synth.gen_quant(DType.Q8_0, 3, rows, cols)
    w = np.frombuffer(w, np.uint8) if isinstance(w, (bytes, bytearray)) else np.asarray(w).view(np.uint8).reshape(-1)
    x = normal(4, (cols,), DType.F32)
    wt, xt = torch.zeros(w.size + 64, dtype=torch.uint8, device="cuda"), torch.zeros(cols + 16, device="cuda")
    yt = torch.zeros(rows + 16, device="cuda")
    wt[:w.size] = torch.from_numpy(w.copy())
    xt[:cols] = x
    with Dev(hip) as d, Imported(hip) as imp:
        hx, hy, ho = imp(xt), imp(yt), d.new(4 * rows)
        exact = hip.import_buffer(wt.data_ptr(), w.size)
        with pytest.raises(YuleGpuError) as e:
            hip.quantized_matmul(exact, hx, hy, rows, cols, DType.Q8_0)
        assert e.value.code == 1 and "slack" in str(e.value)
        hip.free(exact)
        hip.quantized_matmul(imp(wt), hx, hy, rows, cols, DType.Q8_0)
        hip.quantized_matmul(d.up(w), d.up(x), ho, rows, cols, DType.Q8_0)
        want = hip.download(ho, rows)
        assert np.array_equal(yt.cpu().numpy()[:rows], want) and want.any() and not yt[rows:].any()


def test_null_arguments():
    from yule_amd.backend import load_library
    lib, out = load_library(), C.c_uint64()
    assert lib.yule_hip_import_buffer(None, 16, 16, C.byref(out)) == 1 and lib.yule_hip_stream(None, C.byref(C.c_void_p())) == 1


def test_graph_of_the_callers(hip):
    """torch captures its own work and the operators' into one graph on the backend's stream, and replays it between eager
    calls that use the same workspace."""
    say("[import] a graph of torch's")
    be = HipBackend(0)
    heads, kv, hd, prefix, cap, tails, tokens, dt = 8, 2, 64, 900, 30, [30, 4, 11], 2, DType.BF16
    stream = torch.cuda.ExternalStream(be.stream)
    with torch.cuda.stream(stream):
        t = [x.cuda() for x in prefix_inputs(5, heads, kv, hd, prefix, cap, tails, tokens, dt)]
        out, scaled, lens = torch.zeros_like(t[0]), torch.zeros_like(t[0]), ints(tails)
        other = torch.zeros_like(out)
        with Imported(be) as imp:
            q, kp, vp, kt, vt = (imp(x) for x in t)
            hs, ho, hl, hother = imp(scaled), imp(out), imp(lens), imp(other)

            def step():
                torch.mul(t[0], 0.5, out=scaled)
                be.prefix_attn(hs, kp, vp, prefix, kt, vt, hl, cap, ho, len(tails), tokens, heads, kv, hd, dt)
                out.add_(1)

            step()
            torch.cuda.current_stream().synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            for i in range(4):
                t[0].mul_(-1.25)
                lens.copy_(ints([30 - i, 4 + i, 11]))
                out.zero_()
                graph.replay()
                be.prefix_attn(q, kp, vp, prefix, kt, vt, hl, cap, hother, len(tails), tokens, heads, kv, hd, dt)
                got = out.clone()
                step()
                assert torch.equal(bits_of(got), bits_of(out)) and not torch.equal(got, other)
            torch.cuda.current_stream().synchronize()
            del graph
    be.close()
