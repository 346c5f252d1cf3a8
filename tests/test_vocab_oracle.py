"""The 64-bit restatement of the vocabulary's operators against differences."""
from __future__ import annotations

import numpy as np
import pytest

from oracle.vocab import embed_backward, embed_forward, token_loss


@pytest.mark.parametrize("softcap", [0.0, 2.5])
@pytest.mark.parametrize("mean", [True, False])
def test_token_loss_gradients_are_its_differences(softcap, mean):
    rng = np.random.default_rng(3)
    N, D, V = 7, 5, 11
    x, w = rng.standard_normal((N, D)), rng.standard_normal((V, D))
    t = rng.integers(0, V, N)
    t[2] = -1
    weights = rng.uniform(0.5, 1.5, N)
    weights[4] = 0.0
    got = token_loss(x, w, t, weights, softcap, mean, d_total=0.7)
    f = lambda: 0.7 * token_loss(x, w, t, weights, softcap, mean)["total"][0]  # noqa: E731
    h = 1e-5
    for a, d in ((x, got["dx"]), (w, got["dw"])):
        for i in np.ndindex(a.shape):
            keep = a[i]
            a[i] = keep + h
            up = f()
            a[i] = keep - h
            down = f()
            a[i] = keep
            assert abs((up - down) / (2 * h) - d[i]) < 1e-8
    assert np.all(got["dx"][[2, 4]] == 0) and np.all(got["loss"][[2, 4]] == 0)


def test_embedding_gradient_is_the_lookups():
    rng = np.random.default_rng(4)
    N, D, V = 9, 3, 5
    tokens = np.array([0, 4, 4, -1, 2, 5, 0, 0, 2])
    table, dy = rng.standard_normal((V, D)), rng.standard_normal((N, D))
    d = embed_backward(tokens, dy, V, 1.5)
    # linear: <lookup(T), dy> = <T, gradient>
    assert abs((embed_forward(tokens, table, 1.5) * dy).sum() - (table * d).sum()) < 1e-12
    assert np.all(d[[1, 3]] == 0)
    # (the same additions in another order)
    np.testing.assert_allclose(embed_backward(tokens, dy, V, 1.5, before=table), table + d, rtol=0, atol=1e-14)
