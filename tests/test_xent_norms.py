"""The 2-norm bounds of the token loss in fp32 tell planes of operands that are missing
(the restatement on operands of 11 bits) from roundings of fp32."""
import numpy as np
import pytest

from oracle.vocab import token_loss
from tests.xent_norms import errors, norm_bounds

SIZES = [(64, 64, 64), (65, 128, 256), (130, 72, 300), (257, 96, 513), (33, 200, 1000), (300, 544, 130),
         (31, 256, 2049), (100, 1030, 70), (700, 264, 777), (150, 40, 2100), (200, 136, 1000)]


def inputs(N, D, V, seed):
    rng = np.random.default_rng(seed)
    w = (rng.standard_normal((V, D)) * (2.0 / np.sqrt(D))).astype(np.float32)
    t = rng.integers(0, V, N)
    return rng.standard_normal((N, D)).astype(np.float32), w, t


def bits11(a):
    m, e = np.frexp(a.astype(np.float64))
    return np.ldexp(np.round(m * 2048) / 2048, e)


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("N,D,V", SIZES)
def test_a_missing_plane_is_outside(N, D, V, softcap):
    x, w, t = inputs(N, D, V, N + D)
    ref = token_loss(x, w, t, softcap=softcap)
    bounds = norm_bounds(x, w, ref, softcap)
    for a, b in ((bits11(x), w), (x, bits11(w))):
        off = errors(token_loss(a, b, t, softcap=softcap), ref)
        for k in bounds:
            assert off[k] > 2 * bounds[k], (k, off[k] / bounds[k])


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("N,D,V", SIZES)
def test_roundings_of_fp32_are_inside(N, D, V, softcap):
    x, w, t = inputs(N, D, V, N + D)
    rng = np.random.default_rng(1)

    def off(a, bits):
        return a.astype(np.float64) * (1 + 2.0 ** -bits * rng.uniform(-1, 1, a.shape))

    ref = token_loss(x, w, t, softcap=softcap)
    bounds = norm_bounds(x, w, ref, softcap)
    got = errors(token_loss(off(x, 23), off(w, 23), t, softcap=softcap), ref)
    for k in bounds:
        assert got[k] <= bounds[k], (k, got[k] / bounds[k])
