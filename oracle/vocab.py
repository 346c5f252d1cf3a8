"""The operators at the vocabulary's two ends of a training step in 64 bits: the
token embedding and the token loss, with their gradients."""
from __future__ import annotations

import numpy as np


def embed_forward(tokens, table, scale):
    tokens = np.asarray(tokens, np.int64)
    table = np.asarray(table, np.float64)
    out = np.zeros((tokens.size, table.shape[1]))
    inside = (tokens >= 0) & (tokens < table.shape[0])
    out[inside] = scale * table[tokens[inside]]
    return out


def embed_backward(tokens, d_out, V, scale, before=None):
    """d_table, on top of `before`; rows of tokens outside the vocabulary do not count."""
    tokens = np.asarray(tokens, np.int64)
    inside = (tokens >= 0) & (tokens < V)
    d_out = np.asarray(d_out, np.float64)
    d = np.zeros((V, d_out.shape[1])) if before is None else np.array(before, np.float64)
    np.add.at(d, tokens[inside], scale * d_out[inside])
    return d


def token_loss(x, w, targets, weights=None, softcap=0.0, mean=True, d_total=1.0):
    """loss, lse, total, dx, dw, and what tolerances are made of: the rows that take
    part, their logits l, |x| |w| sums and dz."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    targets = np.asarray(targets, np.int64)
    N, V = x.shape[0], w.shape[0]
    weights = np.ones(N) if weights is None else np.asarray(weights, np.float64)
    rows = np.flatnonzero((targets >= 0) & (targets < V) & (weights != 0))
    out = dict(rows=rows, loss=np.zeros(N), lse=np.zeros(N), total=np.zeros(1),
               dx=np.zeros(x.shape), dw=np.zeros(w.shape))
    if rows.size == 0:
        return out
    xs, t, ws = x[rows], targets[rows], weights[rows]
    z = xs @ w.T
    l = softcap * np.tanh(z / softcap) if softcap else z
    top = l.max(axis=1, keepdims=True)
    e = np.exp(l - top)
    s = e.sum(axis=1, keepdims=True)
    lse = (np.log(s) + top)[:, 0]
    at = np.arange(rows.size)
    loss = lse - l[at, t]
    whole = ws.sum() if mean else 1.0
    out["lse"][rows], out["loss"][rows] = lse, loss
    out["total"][0] = (ws * loss).sum() / whole
    g = d_total * ws / whole
    dl = e / s
    # (of the target: minus the others' sum, without the cancellation in p - 1)
    others = dl.copy()
    others[at, t] = 0.0
    dl[at, t] = -others.sum(axis=1)
    dl *= g[:, None]
    dz = dl * (1.0 - (l / softcap) ** 2) if softcap else dl
    out["dx"][rows] = dz @ w
    out["dw"] = dz.T @ xs
    out.update(l=l, z=z, dz=dz, dl=dl, mass=np.abs(xs) @ np.abs(w).T, g=g)
    return out
