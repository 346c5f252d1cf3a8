"""Float64 restatements of the operators around the op's training step: the
residual norm with its gradients (tests pin these by finite differences), the
gradient norm, clipping and AdamW.  With ``absolute=True`` the gradients are
the same sums over absolute values: what an fp32 evaluation's error is
proportional to, term by term."""
from __future__ import annotations

import numpy as np


def _rows(gate, gate_rows, N):
    return np.repeat(gate, gate_rows, axis=0)[:N]


def _ones(v, D):
    return np.ones(D) if v is None else np.asarray(v, np.float64)


def gate_values(gate, sigmoid):
    """The gate's values and their derivatives by what is given."""
    g = np.asarray(gate, np.float64)
    if not sigmoid:
        return g, np.ones_like(g)
    a = 1.0 / (1.0 + np.exp(-g))
    return a, a * (1.0 / (1.0 + np.exp(g)))  # (1 - a loses its digits next to 1)


def resnorm_sum(x, delta, post_scale=None, branch_scale=None, gate=None, gate_rows=1, sigmoid=False,
                post_norm=False, eps=1e-5):
    """(h, the branch's share of it) for x, delta [N, D]; gate [G, 1 or D]."""
    N, D = delta.shape
    z = delta
    if post_norm:
        z = delta / np.sqrt(np.mean(delta * delta, axis=1, keepdims=True) + eps)
    b = _ones(branch_scale, D) * _ones(post_scale, D) * z
    if gate is not None:
        b = b * _rows(gate_values(gate, sigmoid)[0], gate_rows, N)
    return x + b, b


def rms_norm(h, scale=None, eps=1e-5):
    return h / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps) * _ones(scale, h.shape[1])


def resnorm_backward(h, delta, dh, dy, post_scale=None, branch_scale=None, gate=None, gate_rows=1,
                     sigmoid=False, post_norm=False, norm_scale=None, eps=1e-5, absolute=False):
    """Gradients for upstream dh (or None) at h and dy (or None: no norm) at y;
    delta None: no branch.  Returns a dict of dx, d_delta, d_post, d_scale,
    d_gate, d_w."""
    A = np.abs if absolute else (lambda v: v)
    sign = 1.0 if absolute else -1.0
    N, D = (h if h is not None else delta).shape
    t = np.zeros((N, D)) if dh is None else A(dh)
    out = {}
    if dy is not None:
        rn = 1.0 / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
        u = A(dy * _ones(norm_scale, D))
        t = t + rn * u + sign * A(h) * rn ** 3 * np.mean(u * A(h), axis=1, keepdims=True)
        out["d_w"] = np.sum(A(dy * h) * rn, axis=0)
    out["dx"] = t
    if delta is None:
        return out
    rp = np.ones((N, 1))
    if post_norm:
        rp = 1.0 / np.sqrt(np.mean(delta * delta, axis=1, keepdims=True) + eps)
    z = A(delta) * rp
    s, p = A(_ones(branch_scale, D)), A(_ones(post_scale, D))
    q = t * z
    a = 1.0
    if gate is not None:
        value, slope = gate_values(gate, sigmoid)
        a = A(_rows(value, gate_rows, N))
        v = s * p * q
        if gate.shape[1] == 1:
            v = np.sum(v, axis=1, keepdims=True)
        G = gate.shape[0]
        padded = np.zeros((G * gate_rows, v.shape[1])) if G * gate_rows > N else v
        if padded is not v:
            padded[:N] = v
        out["d_gate"] = padded.reshape(G, gate_rows, -1).sum(axis=1) * slope
    column = np.sum(a * q, axis=0)
    out["d_scale"], out["d_post"] = column * p, column * s
    e = t * a * s * p
    if post_norm:
        e = rp * e + sign * A(delta) * rp ** 3 * np.mean(e * A(delta), axis=1, keepdims=True)
    out["d_delta"] = e
    return out


def global_norm(grads):
    return float(np.sqrt(sum(np.sum(np.square(np.asarray(g, np.float64))) for g in grads)))


def clip_coef(norm, max_norm):
    if not np.isfinite(norm) or max_norm <= 0:
        return 1.0
    return min(1.0, max_norm / (norm + 1e-6))


def adamw(p, m, v, g, t, lr, beta1, beta2, eps, decay):
    """One update with the (clipped) gradient g as step t; returns (p, m, v)."""
    p, m, v, g = (np.asarray(a, np.float64) for a in (p, m, v, g))
    m = beta1 * m + (1.0 - beta1) * g
    v = beta2 * v + (1.0 - beta2) * g * g
    update = (m / (1.0 - beta1 ** t)) / (np.sqrt(v / (1.0 - beta2 ** t)) + eps)
    return p - lr * decay * p - lr * update, m, v
