"""The token loss in fp32 against tables some of whose rows are zeros or small: their
gradient is as exact as any other's."""
import numpy as np
import pytest

from mixlab_amd.vocab import TokenLoss
from oracle.vocab import token_loss
from tests.train_testutil import Dev
from tests.xent_norms import rms_bounds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [0.0, 3.0])
@pytest.mark.parametrize("pieces", [False, True])
@pytest.mark.parametrize("N,D,V", [(520, 64, 300), (40, 72, 4100), (520, 40, 16500), (300, 64, 50257)])
def test_gradients_of_small_rows(gpu_lib, N, D, V, pieces, softcap, monkeypatch):
    """The logits are of size one, so that every entry's share is about 1 / V and the others'
    gradients are far below the target's."""
    if pieces:
        monkeypatch.setenv("MXM_XENT_PIECE_BYTES", "1")
    rng = np.random.default_rng(V)
    x = rng.standard_normal((N, D)).astype(np.float32)
    w = (rng.standard_normal((V, D)) * 0.1).astype(np.float32)
    groups = {"zero": 0.0, "2^-30": 2.0 ** -30, "2^-12": 2.0 ** -12, "2^-6": 2.0 ** -6, "2^-3": 2.0 ** -3, "one": 1.0}
    for i, f in enumerate(groups.values()):
        w[i::len(groups)] *= np.float32(f)
    t = rng.integers(0, V, N).astype(np.int32)
    dx_, dw_, dt, gx, gw = Dev(x), Dev(w), Dev(t, "int32"), Dev.out((N, D)), Dev.out((V, D))
    with TokenLoss(V, D, N, dtype="fp32", softcap=softcap) as h:
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr)
        h.synchronize()
    ref = token_loss(x, w, t, softcap=softcap)
    # (2^-36 of a row's largest: planes that end at 2^-40, the slack of four bits)
    bound = rms_bounds(x, w, ref, softcap, 2.0 ** -36)
    dx, dw = gx.get(), gw.get()
    others = ~np.isin(np.arange(V), t)
    for i, name in enumerate(groups):
        rows = t % len(groups) == i
        off = np.linalg.norm(dx[rows] - ref["dx"][rows]) / np.linalg.norm(bound["dx"][rows])
        assert off <= 1, ("dx, target", name, off)
        for what, is_in in (("no target", others), ("target", ~others)):
            s = np.flatnonzero(is_in & (np.arange(V) % len(groups) == i))
            if len(s):
                off = np.linalg.norm(dw[s] - ref["dw"][s]) / np.linalg.norm(bound["dw"][s])
                assert off <= 1, ("dw", what, name, off)
