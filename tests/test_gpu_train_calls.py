"""Calls on residual norms and gradient sets in orders, at values and over
buffers that a program can come to."""
import numpy as np
import pytest

from oracle import train as ot
from tests.test_gpu_train_streams import Graph
from tests.train_testutil import Dev, close

pytestmark = pytest.mark.gpu


def test_replayed_update_after_a_bind_without_params(gpu_lib):
    """A captured AdamW step reads the pointers bound last: with none for params it
    updates nothing, and goes on once they are bound again."""
    from mixlab_amd.train import GradientSet

    sizes = [1000, 0, 3]
    rng = np.random.default_rng(0)
    with GradientSet(sizes) as s:
        g, p, m, v = ([Dev(rng.random(n, dtype=np.float32)) for n in sizes] for _ in range(4))
        ptrs = [[d.ptr for d in one] for one in (g, p, m, v)]
        step, skipped, norm = Dev(np.zeros(1, np.int64), "int64"), Dev.out((1,), np.int32), Dev.out((1,))

        def state():
            s.synchronize()
            return [d.get() for one in (p, m, v) for d in one]

        s.bind(ptrs[0], params=ptrs[1], m=ptrs[2], v=ptrs[3])
        graph = Graph(gpu_lib, s.stream(), lambda: s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, 0.0, step.ptr,
                                                           norm.ptr, skipped.ptr))
        graph.replay()
        once = state()
        assert step.get()[0] == 1 and skipped.get()[0] == 0
        s.bind(ptrs[0])
        graph.replay()
        for a, b in zip(state(), once):
            assert np.array_equal(a, b)
        assert step.get()[0] == 1 and skipped.get()[0] == 1
        close(norm.get(), [ot.global_norm([d.get() for d in g])], 0, "fp32", "norm")
        s.bind(ptrs[0], params=ptrs[1], m=ptrs[2], v=ptrs[3])
        graph.replay()
        assert not np.array_equal(state()[0], once[0])
        assert step.get()[0] == 2 and skipped.get()[0] == 0
        graph.close()
