"""Bounds of the token loss's errors in the 2-norm, for fp32 operands: what fp32 precision
means for results that elementwise worst cases are far too wide for."""
import numpy as np

from tests.train_testutil import U32


def rms_bounds(x, w, ref, softcap=0.0, floor=0.0):
    """Of loss, lse, dx and dw of the rows that take part (x and ref's), element by element,
    for 2-norms over many of them.  floor: what the logits' gradient is off by at least, of
    its row's largest.

    Roundings of different elements are independent: they add up by squares.  A logit's
    error: of each product of elements the operands' half steps of 2^-23 and the product of
    the small planes that is left out, below 2^-22 (together below 4 U32 of the products'
    root sum of squares); a step (2 U32, 0.3 of it at its root mean square, taken as U32 / 2)
    of the partial sums for each of three planes' additions of 16 products; an exponential's
    argument of at most 2^4 or the logit's size.  Of a row's errors the softmax takes the sum
    weighted by the shares, common to the row."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    z, dz, dl, g = ref["z"], np.abs(ref["dz"]), np.abs(ref["dl"]), np.abs(ref["g"])
    rows = ref["rows"]
    root = np.sqrt(x ** 2 @ (w ** 2).T)
    el = U32 * (4 * root + np.sqrt(3 * x.shape[1] / 16) / 2 * (root + np.abs(z)) + np.abs(z) + 8) + 4 * U32 * softcap
    share = np.divide(dl, g[:, None], out=np.zeros_like(dl), where=g[:, None] > 0)
    common = np.sqrt(((share * el) ** 2).sum(axis=1))
    few = U32 * (8 + 2 * np.abs(ref["lse"][rows]) + 4 * softcap)
    p = np.exp(ref["l"] - ref["lse"][rows][:, None])
    rel = np.sqrt(el ** 2 + common[:, None] ** 2) + 8 * U32
    if softcap:
        rel = rel + 2 * el / softcap + U32 * (4 * np.abs(z) / softcap + 8)
    edz = dz * rel + floor * dl.max(axis=1, keepdims=True)
    dx = np.sqrt(edz ** 2 @ w ** 2) + 8 * U32 * np.sqrt(dz ** 2 @ w ** 2) + 4 * U32 * np.abs(ref["dx"][rows])
    dw = np.sqrt((edz ** 2).T @ x ** 2) + 8 * U32 * np.sqrt((dz ** 2).T @ x ** 2) + 4 * U32 * np.abs(ref["dw"])
    return {"loss": common + few + 4 * U32 * ref["loss"][rows],
            "lse": np.sqrt(((p * el) ** 2).sum(axis=1)) + few, "dx": dx, "dw": dw}


def norm_bounds(x, w, ref, softcap=0.0):
    """The same as 2-norms over all."""
    return {k: np.linalg.norm(v) for k, v in rms_bounds(x, w, ref, softcap).items()}


def errors(got, ref):
    """2-norms of what the results (of the rows that take part) are off by."""
    rows = ref["rows"]
    want = {"loss": ref["loss"][rows], "lse": ref["lse"][rows], "dx": ref["dx"][rows], "dw": ref["dw"]}
    return {k: np.linalg.norm(np.asarray(got[k], np.float64) - want[k]) for k in want}
