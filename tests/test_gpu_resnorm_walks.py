"""Residual norms over so many rows that a thread walks several: the forward's
rows a thread, and the backward's chunks of several whole groups of gate rows.
Row results are compared on a sample (the first and last rows and 300 between),
the column sums and the gates' gradients whole.  Tolerances as in
test_gpu_resnorm."""
import numpy as np
import pytest

from oracle import train as ot
from tests.test_gpu_resnorm import _case, _col_c, _handle, _row_c, run_backward, run_forward
from tests.train_testutil import U32, as_kept, close

pytestmark = pytest.mark.gpu

TYPES = {"fp32": {}, "bf16": dict(stream="bf16", delta="bf16", out="bf16", grad="bf16")}


def _sample(N, seed):
    between = np.random.default_rng(seed).integers(0, N, 300)
    return np.unique(np.concatenate([np.arange(20), between, np.arange(N - 40, N)]))


# rows in a workgroup (two or four a thread), in waves, side by side in a wave; odd widths too
WALKS = [(8203, 2048), (8197, 1030), (8201, 4097), (35003, 520), (33001, 769), (70001, 100), (140003, 64),
         (133001, 37)]


@pytest.mark.parametrize("N,D", WALKS)
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("gate,gate_rows,sigmoid", [("row", 1, True), ("row", 3, False), ("channel", 700, True)])
def test_forward_walks(gpu_lib, N, D, types, gate, gate_rows, sigmoid):
    c = dict(TYPES[types], gate=gate, gate_rows=gate_rows, sigmoid=sigmoid)
    v = _case(N + D, 1, D, **dict(c, gate=None))
    rng = np.random.default_rng(N)
    for k, size, kept in (("x", 1.0, "stream"), ("delta", 0.3, "delta")):
        v[k] = as_kept(rng.standard_normal((N, D), dtype=np.float32) * np.float32(size), c.get(kept, "fp32"))
    v["gate"] = rng.standard_normal((-(-N // gate_rows), D if gate == "channel" else 1), dtype=np.float32)
    with _handle(N, D, backward=False, **c) as r:
        h, y = (t.get() for t in run_forward(v, N, D, handle=r, **c))
    at = _sample(N, D)
    f = lambda k: v[k][at].astype(np.float64)  # noqa: E731
    want, share = ot.resnorm_sum(f("x"), f("delta"), v["post_scale"], v["branch_scale"],
                                 v["gate"][at // gate_rows], 1, sigmoid, True)
    close(h[at], want, _row_c(D) * np.abs(share) + U32 * np.abs(want), types, "h")
    want = ot.rms_norm(h[at].astype(np.float64), v["norm_scale"])
    close(y[at], want, _row_c(D) * np.abs(want), types, "y")
    assert np.isfinite(h).all() and np.isfinite(y).all()


# (rows, channels, gate rows): chunks of two groups or more, the last group short
GROUPS = [(8501, 260, 2), (13001, 260, 3), (50001, 64, 2), (33000, 101, 2), (2101, 2048, 2), (4501, 2048, 4),
          (3101, 1030, 2), (9001, 900, 2)]


@pytest.mark.parametrize("N,D,gate_rows", GROUPS)
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("gate,sigmoid", [("row", True), ("channel", False), ("channel", True)])
def test_backward_chunks_of_groups(gpu_lib, N, D, gate_rows, types, gate, sigmoid):
    c = dict(TYPES[types], gate=gate, gate_rows=gate_rows, sigmoid=sigmoid)
    v = _case(N + D + gate_rows, N, D, **c)
    with _handle(N, D, **c) as r:
        got = run_backward(v, N, D, handle=r, **c)
    f = lambda k: v[k].astype(np.float64)  # noqa: E731
    args = (f("h"), f("delta"), f("dh"), f("dy"), v["post_scale"], v["branch_scale"], v["gate"], gate_rows,
            sigmoid, True, v["norm_scale"])
    want, size = ot.resnorm_backward(*args), ot.resnorm_backward(*args, absolute=True)
    assert set(got) == set(want)
    for k in got:
        if k in ("dx", "d_delta"):
            close(got[k], want[k], _row_c(D) * size[k], types, k)
        else:
            close(got[k], want[k], _col_c(N, D) * size[k], "fp32", k)
