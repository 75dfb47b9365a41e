"""The backend's workspace where graphs were captured with it and a larger one
cannot be had."""
import numpy as np
import pytest
import torch

from test_batch_gpu import Dev, bits_of, prefix_inputs, run_prefix, say
from yule_amd import DType
from yule_amd.backend import HipBackend, YuleGpuError

pytestmark = pytest.mark.gpu

SHAPE = (32, 8, 128, 4096, 0, [0] * 64, 1)   # 16 chunks of 64 x 32 rows of 128 f32 sums, and a little: 17 MiB


def test_growth_that_fails(monkeypatch):
    """A call that finds no room takes nothing with it: the graph's workspace serves the next calls, and captures of them take
    no memory each."""
    say("[workspace] growth that fails, between captures")
    heads, kv, hd, prefix, cap, lens, tokens = SHAPE
    be, dt = HipBackend(0), DType.BF16
    x = prefix_inputs(1, heads, kv, hd, prefix, cap, lens, tokens, dt)
    more = prefix_inputs(2, heads, kv, hd, 2 * prefix, cap, lens, tokens, dt)
    with Dev(be) as d:
        want = run_prefix(be, d, *x, lens, cap, tokens, heads, kv, hd, dt)
        out, big = d.new(want.numel() * 2), d.new(want.numel() * 2)
        ln = d.up(np.array(lens, np.uint32))
        args = [(d.up(q), d.up(kp), d.up(vp), kp.shape[0], None, None, ln, cap, o, len(lens), tokens, heads, kv, hd, dt)
                for (q, kp, vp, _, _), o in ((x, out), (more, big))]
        free = []
        for _ in range(6):
            be.capture_begin()
            be.prefix_attn(*args[0])
            be.capture_end()
            with monkeypatch.context() as m:
                m.setenv("YULE_WORKSPACE_LIMIT_MB", "1")
                with pytest.raises(YuleGpuError) as e:
                    be.prefix_attn(*args[1])
                assert e.value.code == 4
            be.copy_to_device(np.zeros(want.numel(), np.uint16), out)
            be.prefix_attn(*args[0])   # eagerly, and by the graph
            eager = d.down(out, tuple(want.shape), dt)
            be.copy_to_device(np.zeros(want.numel(), np.uint16), out)
            be.capture_replay()
            got = d.down(out, tuple(want.shape), dt)
            assert torch.equal(bits_of(eager), bits_of(want)) and torch.equal(bits_of(got), bits_of(want))
            free.append(torch.cuda.mem_get_info()[0])
        assert free[0] - free[-1] < 16 << 20, free
        be.prefix_attn(*args[1])       # there is room now
        be.synchronize()
        be.capture_replay()            # with its own workspace still
        got = d.down(out, tuple(want.shape), dt)
        assert torch.equal(bits_of(got), bits_of(want))
    be.close()
