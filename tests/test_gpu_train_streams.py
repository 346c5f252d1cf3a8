"""Handles on shared streams, several handles and threads at once, and calls
captured into a HIP graph and replayed."""
import ctypes
import threading

import numpy as np
import pytest

from mixlab_amd import _lib
from oracle import train as ot
from tests.train_testutil import U32, Dev, close

pytestmark = pytest.mark.gpu


def _data(seed, N, D):
    rng = np.random.default_rng(seed)
    return {k: rng.standard_normal((N, D), dtype=np.float32) for k in ("x", "delta", "dh", "dy")}


def _want_h(v):
    return ot.resnorm_sum(v["x"].astype(np.float64), v["delta"].astype(np.float64), post_norm=True)[0]


def test_shared_stream_outlives_its_first_handle(gpu_lib):
    from mixlab_amd.op import MoEFeedForward
    from mixlab_amd.train import GradientSet, ResidualNorm

    N, D = 33, 96
    v = _data(0, N, D)
    op = MoEFeedForward([1, N, D, 2, 1, 0, 64, 0])
    r = ResidualNorm(D, N, out_dtype="fp32", post_norm=True, share=op)
    s = GradientSet([N * D], share=r)
    assert r.stream() == s.stream() != 0
    op.close()
    x, d, h, y, n = Dev(v["x"]), Dev(v["delta"]), Dev.out((N, D)), Dev.out((N, D)), Dev.out((1,))
    s.bind([h.ptr])
    r.forward(N, x.ptr, d.ptr, h.ptr, y.ptr)
    s.norm(n.ptr)  # after the forward, without a wait
    r.close()
    s.synchronize()
    want = _want_h(v)
    close(n.get(), [ot.global_norm([want])], (D / 64 + 40) * U32 * np.linalg.norm(want), "fp32", "norm")
    s.close()


def test_threads(gpu_lib):
    """Distinct handles from several threads at once."""
    from mixlab_amd.train import GradientSet, ResidualNorm

    N, D, bad = 200, 1024, []

    def work(seed):
        try:
            v = _data(seed, N, D)
            with ResidualNorm(D, N, out_dtype="fp32", post_norm=True) as r, GradientSet([N * D]) as s:
                x, d = Dev(v["x"]), Dev(v["delta"])
                h, y, n = Dev.out((N, D)), Dev.out((N, D)), Dev.out((1,))
                s.bind([x.ptr])
                for _ in range(20):
                    r.forward(N, x.ptr, d.ptr, h.ptr, y.ptr)
                    s.norm(n.ptr)
                r.synchronize()
                s.synchronize()
                want = _want_h(v)
                close(h.get(), want, (D / 64 + 40) * U32 * (np.abs(want) + np.abs(v["x"])), "fp32", "h")
                close(n.get(), [ot.global_norm([v["x"]])], 0, "fp32", "norm")
        except BaseException as e:
            bad.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad[0]


class Graph:
    """A graph captured on a handle's stream, through the HIP runtime that the
    library is linked to."""

    def __init__(self, lib, stream, calls):
        self.lib, self.stream = lib, ctypes.c_void_p(stream)
        graph, self.exe = ctypes.c_void_p(), ctypes.c_void_p()
        assert lib.hipStreamBeginCapture(self.stream, 0) == 0
        calls()
        assert lib.hipStreamEndCapture(self.stream, ctypes.byref(graph)) == 0
        assert lib.hipGraphInstantiate(ctypes.byref(self.exe), graph, None, None, ctypes.c_size_t(0)) == 0
        assert lib.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.lib.hipGraphLaunch(self.exe, self.stream) == 0

    def close(self):
        assert self.lib.hipGraphExecDestroy(self.exe) == 0


def test_captured_and_replayed(gpu_lib):
    """Forward, backward, clip and AdamW in one graph, replayed with new data in the
    same buffers and eager calls between, each replay against the eager result."""
    from mixlab_amd.train import GradientSet, ResidualNorm

    N, D = 70, 260
    sizes = (D, N * D, 0, 5)
    rng = np.random.default_rng(0)
    with ResidualNorm(D, N, out_dtype="fp32", post_norm=True, gate="channel", gate_rows=30) as r, \
            GradientSet(sizes, decay=[0, 1, 1, 1], share=r) as s:
        inp = {k: Dev.out((N, D)) for k in ("x", "delta", "dh", "dy")}
        out = {k: Dev.out((N, D)) for k in ("h", "y", "dx", "dd")}
        out.update({k: Dev.out((D,)) for k in ("dp", "ds", "dw")}, dg=Dev.out((3, D)), norm=Dev.out((1,)))
        vec = {k: Dev(rng.random(D, dtype=np.float32) + 0.5) for k in ("post", "scale", "w")}
        gate, extra = Dev(rng.random((3, D), dtype=np.float32)), Dev(rng.random(5, dtype=np.float32))
        step = Dev(np.zeros(1, np.int64), "int64")
        state = {k: [Dev(np.zeros(n, np.float32)) for n in sizes] for k in ("p", "m", "v")}
        clipped = [Dev.out((n,)) for n in sizes]
        s.bind([out["dw"].ptr, out["dx"].ptr, 0, extra.ptr], [c.ptr for c in clipped],
               *[[b.ptr for b in state[k]] for k in ("p", "m", "v")])

        def calls():
            r.forward(N, inp["x"].ptr, inp["delta"].ptr, out["h"].ptr, out["y"].ptr, vec["post"].ptr,
                      vec["scale"].ptr, gate.ptr, vec["w"].ptr)
            r.backward(N, out["h"].ptr, inp["delta"].ptr, inp["dh"].ptr, inp["dy"].ptr, out["dx"].ptr,
                       out["dd"].ptr, vec["post"].ptr, vec["scale"].ptr, gate.ptr, vec["w"].ptr,
                       out["dp"].ptr, out["ds"].ptr, out["dg"].ptr, out["dw"].ptr)
            s.clip(0.5, out["norm"].ptr)
            s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, 0.5, step.ptr, out["norm"].ptr)

        def fill(seed):
            g = np.random.default_rng(seed)
            for b in inp.values():
                b.put(g.standard_normal((N, D), dtype=np.float32))
            for k in ("p", "m", "v"):
                for b in state[k]:
                    b.put(g.random(b.size, dtype=np.float32))
            step.put(np.full(1, seed, np.int64))

        def results():
            r.synchronize()
            everything = list(out.values()) + clipped + [b for k in ("p", "m", "v") for b in state[k]]
            return [b.get() for b in everything + [step]]

        fill(0)
        graph = Graph(gpu_lib, r.stream(), calls)
        for seed in (1, 2, 3):
            fill(seed)
            calls()  # eager
            want = results()
            fill(seed + 10)
            calls()
            other = results()
            fill(seed)
            graph.replay()
            got = results()
            assert not np.array_equal(other[0], want[0])
            for a, b in zip(got, want):
                assert np.array_equal(a, b)
        graph.close()
