"""The float64 restatement of the residual norm's gradients against central
differences of its forward, and of AdamW against its definition's limits (CPU)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import train as ot


@pytest.mark.parametrize("post_norm", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("gate,gate_rows,sigmoid", [(None, 1, False), ("row", 1, True),
                                                    ("row", 3, False), ("channel", 1, False),
                                                    ("channel", 3, True)])
def test_gradients_match_differences(post_norm, norm, gate, gate_rows, sigmoid):
    N, D, eps = 7, 5, 1e-2
    rng = np.random.default_rng(5)
    v = dict(x=rng.standard_normal((N, D)), delta=rng.standard_normal((N, D)),
             post=1 + 0.3 * rng.standard_normal(D), scale=1 + 0.3 * rng.standard_normal(D),
             w=1 + 0.3 * rng.standard_normal(D))
    if gate:
        v["gate"] = rng.standard_normal((-(-N // gate_rows), D if gate == "channel" else 1))
    dh, dy = rng.standard_normal((N, D)), rng.standard_normal((N, D))

    def loss(v):
        h, _ = ot.resnorm_sum(v["x"], v["delta"], v["post"], v["scale"], v.get("gate"), gate_rows,
                              sigmoid, post_norm, eps)
        out = np.sum(h * dh)
        return out + (np.sum(ot.rms_norm(h, v["w"], eps) * dy) if norm else 0.0)

    h, _ = ot.resnorm_sum(v["x"], v["delta"], v["post"], v["scale"], v.get("gate"), gate_rows,
                          sigmoid, post_norm, eps)
    got = ot.resnorm_backward(h, v["delta"], dh, dy if norm else None, v["post"], v["scale"],
                              v.get("gate"), gate_rows, sigmoid, post_norm, v["w"], eps)
    names = dict(x="dx", delta="d_delta", post="d_post", scale="d_scale", w="d_w", gate="d_gate")
    step = 1e-5
    for k, arr in v.items():
        if k == "w" and not norm:
            continue
        for i in [tuple(rng.integers(0, s) for s in arr.shape) for _ in range(8)]:
            old = arr[i]
            arr[i] = old + step
            up = loss(v)
            arr[i] = old - step
            down = loss(v)
            arr[i] = old
            # (third derivatives of these O(1) formulas times step^2, and 1e-15 / step)
            assert abs((up - down) / (2 * step) - got[names[k]][i]) <= 1e-7 * (1 + abs(got[names[k]][i])), k


def test_adamw_first_step_is_a_signed_step():
    """From zero state the bias-corrected update is g / (|g| + eps): the step is lr
    against the gradient's sign, and decay is taken from the value before it."""
    p, g = np.array([1.0, -2.0, 0.5]), np.array([3.0, -1e-3, 0.0])
    q, m, v = ot.adamw(p, np.zeros(3), np.zeros(3), g, 1, 0.1, 0.9, 0.999, 1e-12, 0.5)
    np.testing.assert_allclose(q, p - 0.05 * p - 0.1 * np.sign(g), rtol=1e-8)
    np.testing.assert_allclose(m, 0.1 * g)
    np.testing.assert_allclose(v, 0.001 * g * g)


def test_clipping():
    assert ot.global_norm([[3.0], [4.0]]) == 5.0
    assert ot.clip_coef(5.0, 10.0) == 1.0 and abs(ot.clip_coef(5.0, 1.0) - 0.2) < 1e-6
    assert ot.clip_coef(float("inf"), 1.0) == 1.0
