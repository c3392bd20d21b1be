"""Page table calls captured more often than the library has counters for calls of
several workgroups: those behind are done by one.  Last of the files, as what is
captured keeps its counter for good."""
import numpy as np
import pytest

import kvad_amd as K
import test_gpu_step as T

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_more_captured_calls_than_counters():
    stream, ctx = torch.cuda.Stream(), K.Context(0)
    torch.cuda.synchronize()
    try:
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            t = T.Tables(ctx, 64, 60, 32, 3000)
            rows, keep = (torch.full((64,), v, dtype=torch.int32, device="cuda") for v in (0, -1))
            pos, slot = (torch.zeros(4000, dtype=d, device="cuda") for d in (torch.int32, torch.int64))
            assert t.step([1] * 64, 4000) == 0  # the context's own counter
        torch.cuda.synchronize()
        for n in (1 << 14, 1):  # all that there are, never replayed; then one more of each call
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                for _ in range(n):
                    t.t.release_dev(ctx, keep.data_ptr())
                    t.t.step_dev(ctx, rows.data_ptr(), 4000, pos.data_ptr(), slot.data_ptr())
            torch.cuda.synchronize()
        rng = np.random.default_rng(4)
        with torch.cuda.stream(stream):
            for i in range(4):
                k = [n // 2 if s % 2 and i else -1 for s, n in enumerate(t.len)]
                r = [int(x) for x in rng.integers(0, 62, 64)]
                keep.copy_(torch.tensor(k))
                rows.copy_(torch.tensor(r))
                g.replay()
                for s in reversed(range(64)):
                    if 0 <= k[s] < t.len[s]:
                        for j in reversed(range(t.pages_of(k[s]), t.pages_of(t.len[s]))):
                            t.free.append(t.pages[s][j])
                            t.pages[s][j] = -1
                        t.len[s] = k[s]
                t.expect(r, 4000)
                t.check()
                assert pos.cpu().tolist() == t.position and slot.cpu().tolist() == t.slot
                # beside it the context's own calls, of several workgroups still
                assert t.step([3] * 64, 4000) == 0
        del g
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(None)
        ctx.close()
