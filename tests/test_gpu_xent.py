"""The token loss on the device against its 64-bit restatement: rows that take no
part (whatever they hold), odd sizes, alignments and types, one row and many,
pieces of the rows, extreme logits."""
from __future__ import annotations

import numpy as np
import pytest

from mixlab_amd import _lib
from mixlab_amd.vocab import TokenLoss
from oracle.vocab import token_loss
from train_testutil import U32, UBF, Dev, as_kept, close

pytestmark = pytest.mark.gpu


def tolerances(x, w, ref, dtype, softcap, V):
    """Bounds of loss, lse, dx and dw (of the rows that take part), from the roundings.

    A logit is a sum of D products in fp32, of which each partial sum may lose a whole
    step (2 U32) in the matrix cores.  Under fp32 a row of an operand is two fp16 planes
    of 11 bits each, in units of which its largest element is over 2^14: 2^-23 of an
    element (2 U32), or half a subnormal step, 2^-25 and so 2^-39 of the row's largest;
    three products of planes are summed, and the fourth, left out, is below 2^-22 (4 U32).
    An exponential's argument l - ref is rounded once (U32 |l|), the exponential and
    each of the sum's additions once or twice."""
    D = x.shape[1]
    fp32 = dtype == "fp32"
    aw, ax = np.abs(w), np.abs(x)
    xtop, wtop = ax.max(axis=1, keepdims=True), aw.max(axis=1, keepdims=True)
    low = 2.0 ** -39
    dz, dl = np.abs(ref["dz"]), np.abs(ref["dl"])
    # |g| times the others' share bounds a row's |dl|; the target's is that
    most = dl.max(axis=1, keepdims=True)
    if fp32:
        # the least exponent of a row of the table: smaller ones are taken down to it (at
        # most: it has some slack)
        others = np.where(ref["dl"] * ref["g"][:, None] > 0, dz, 0.0)
        least = np.divide(others * wtop.T, most, out=np.zeros_like(dl), where=most > 0).max()
        wtop = np.maximum(wtop, least)
    el = (2 * (D + 8) * (3 if fp32 else 1) + (8 if fp32 else 4)) * U32 * ref["mass"]
    if fp32:
        el = el + low * (xtop * aw.sum(axis=1) + ax.sum(axis=1, keepdims=True) * wtop.T)
    if softcap:
        el = el + 8 * U32 * softcap
    # an entry whose logit is over 60 below the largest, whatever its error, has a share
    # below 2^-86
    alive = ref["l"] + 2 * el > (ref["l"] - 2 * el).max(axis=1, keepdims=True) - 60
    size = np.where(alive, np.abs(ref["l"]), 0.0).max(axis=1, keepdims=True)
    top = np.where(alive, el, 0.0).max(axis=1, keepdims=True)
    steps = U32 * (8 * size + 2 * (V / 64 + 160))
    # (the target's own logit is in the loss; of lse it is not asked for)
    at_target = np.where(ref["dl"] * ref["g"][:, None] > 0, 0.0, el + 8 * U32 * np.abs(ref["l"])).max(axis=1)
    row = (2 * top + steps)[:, 0] + at_target
    ep = (2 * top + steps) * 1.1            # of p, relative
    rounding = 8 * U32 if fp32 else UBF + UBF / 4
    edz = dz * (ep + rounding) + most * 2.0 ** -86
    if fp32:
        # dz is kept in planes too, in units of the row's largest |dz| times its row of the
        # table, or of the largest |dz| times the least exponent (a power of two from each:
        # within a factor of 8; the slack of four bits); half a subnormal step is 2^-39 of them
        scale = np.maximum((dz * wtop.T).max(axis=1, keepdims=True), most * least)
        scale = np.where(scale > 0, scale, most)  # (a table of zeros)
        edz = edz + low * 8 * 16 * scale / np.where(wtop.T > 0, wtop.T, 1.0)
    else:
        # p is kept in fp16 between its two passes, in units of which the largest of a
        # block of the vocabulary is over 2^14: half a step of fp16's subnormal numbers,
        # 2^-25, is 2^-39 of that largest one, which is at most the row's largest p
        edz = edz + most * low
    if softcap:                             # of 1 - (l / cap)^2
        edz = edz + dl * (2 * el / softcap + 16 * U32)
    per = 2 * (3 if fp32 else 1)
    N = x.shape[0]
    bx = edz @ aw + per * (V + 64) * U32 * ((dz + edz) @ aw)
    bw = edz.T @ ax + per * (N + 64) * U32 * ((dz + edz).T @ ax)
    if fp32:
        bx = bx + dz @ (4 * U32 * aw + low * wtop)
        # dw's rows of x share one exponent, set by the largest of those units times row of x
        share = np.divide(dz, scale, out=np.zeros_like(dz), where=scale > 0)
        bw = bw + dz.T @ (4 * U32 * ax) + (low * 8 * (scale * xtop).max()) * share.sum(axis=0)[:, None]
    return row, bx, bw


def check(x, w, t, weights=None, dtype="bf16", dx_dtype="fp32", dw_dtype="fp32", softcap=0.0, mean=True,
          d_total=1.0, shift=0, max_rows=None, calls=1, handle=None, want_dx=True, want_dw=True):
    N, D = x.shape
    V = w.shape[0]
    dx_, dw_ = Dev(x, dtype, shift), Dev(w, dtype, shift)
    dt = Dev(t.astype(np.int32), "int32")
    dr = None if weights is None else Dev(weights)
    out = {k: Dev.out(s) for k, s in (("loss", (N,)), ("lse", (N,)), ("total", (1,)))}
    fwd = {k: Dev.out(s) for k, s in (("loss", (N,)), ("lse", (N,)), ("total", (1,)))}
    gx, gw = Dev.out((N, D), dx_dtype, shift), Dev.out((V, D), dw_dtype, shift)
    h = handle or TokenLoss(V, D, max_rows or N, dtype=dtype, dx_dtype=dx_dtype, dw_dtype=dw_dtype,
                            softcap=softcap, mean=mean)
    ptrs = lambda o: {k: v.ptr for k, v in o.items()}  # noqa: E731
    bits = None
    for _ in range(calls):
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr if want_dx else 0, dw=gw.ptr if want_dw else 0,
                   row_weights=dr.ptr if dr else 0, d_total=d_total, **ptrs(out))
        h.forward(N, dx_.ptr, dw_.ptr, dt.ptr, row_weights=dr.ptr if dr else 0, **ptrs(fwd))
        h.synchronize()
        now = [out[k].get() for k in out] + [gx.get(), gw.get()]
        if bits is not None:
            for a, b in zip(bits, now):
                np.testing.assert_array_equal(a, b)
        bits = now
    if handle is None:
        h.close()
    took = np.flatnonzero((t >= 0) & (t < V) & (True if weights is None else weights != 0))
    clean = np.zeros_like(x)
    clean[took] = x[took]
    ref = token_loss(clean, w, t, weights, softcap, mean, d_total)
    left = np.setdiff1d(np.arange(N), took)
    for o in (out, fwd):
        assert np.all(o["loss"].get()[left] == 0) and np.all(o["lse"].get()[left] == 0)
    if took.size == 0:
        assert out["total"].get()[0] == 0 and fwd["total"].get()[0] == 0
        assert not want_dx or np.all(gx.get() == 0)
        assert not want_dw or np.all(gw.get() == 0)
        return
    row, bx, bw = tolerances(clean[took], w, ref, dtype, softcap, V)
    for o in (out, fwd):
        close(o["loss"].get()[took], ref["loss"][took], row, "fp32", "loss")
        close(o["lse"].get()[took], ref["lse"][took], row, "fp32", "lse")
        part = np.abs(ref["g"] / d_total if d_total else ref["g"])
        if d_total:
            close(o["total"].get(), ref["total"], (part * (row + 2 * U32 * np.abs(ref["loss"][took]))).sum(),
                  "fp32", "total")
    if want_dx:
        got = gx.get()
        close(got[took], ref["dx"][took], bx, dx_dtype, "dx")
        assert np.all(got[left] == 0)
        near(got, ref["dx"], dtype, dx_dtype, bx, "dx")
    if want_dw:
        got = gw.get()
        close(got, ref["dw"], bw, dw_dtype, "dw")
        near(got, ref["dw"], dtype, dw_dtype, bw, "dw")


def near(got, want, dtype, kept, bound, what):
    """The 2-norm of the error.  Roundings to bf16 are independent and each off by at most
    half a step, 0.58 of it at its root mean square; two of them (the logits' gradient
    and the result) and the sums stay below one and a half half steps."""
    if dtype == "bf16" or kept == "bf16":
        off, size = np.linalg.norm(got - want), np.linalg.norm(want)
        assert off <= 1.5 * UBF * size + 1e-30, (what, off / size)


def inputs(N, D, V, dtype, seed, size=1.0, pad=0.0):
    rng = np.random.default_rng(seed)
    w = as_kept(rng.standard_normal((V, D)) * (2.0 * size / np.sqrt(D)), dtype)
    t = rng.integers(0, V, N).astype(np.int64)
    x = rng.standard_normal((N, D))
    norm = (w[t].astype(np.float64) ** 2).sum(axis=1, keepdims=True) + 1e-30
    x = as_kept(x + w[t] * (rng.random((N, 1)) * 8.0 * size / norm), dtype)
    if pad:
        out = rng.random(N) < pad
        t[out] = rng.choice(np.array([-1, -100, V, 2 ** 31 - 1, -2 ** 31]), out.sum())
        x[out] = np.nan
    return x, w, t


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V", [
    (1, 64, 100), (1, 1, 1), (1, 7, 2), (3, 65, 257), (64, 64, 64), (65, 128, 256), (130, 72, 300),
    (257, 96, 513), (33, 200, 1000), (300, 544, 130), (512, 33, 40), (31, 256, 2049), (100, 1030, 70),
    (700, 264, 777),
])
def test_sizes(gpu_lib, N, D, V, dtype):
    x, w, t = inputs(N, D, V, dtype, N + D + V)
    check(x, w, t, dtype=dtype, dx_dtype=dtype, dw_dtype=dtype, calls=2)


@pytest.mark.parametrize("dtype,dx,dw,softcap,mean,weighted,pad,shift", [
    ("bf16", "fp32", "fp32", 0.0, True, False, 0.3, 0),
    ("bf16", "bf16", "fp32", 30.0, True, True, 0.0, 0),
    ("bf16", "fp32", "bf16", 5.0, False, True, 0.5, 1),
    ("fp32", "fp32", "fp32", 30.0, False, True, 0.3, 0),
    ("fp32", "bf16", "bf16", 0.0, True, True, 0.9, 1),
    ("fp32", "fp32", "bf16", 2.0, True, False, 0.0, 3),
])
@pytest.mark.parametrize("N,D,V", [(200, 64, 384), (321, 136, 1001), (45, 37, 90)])
def test_forms(gpu_lib, N, D, V, dtype, dx, dw, softcap, mean, weighted, pad, shift):
    x, w, t = inputs(N, D, V, dtype, 7 * N + V, pad=pad)
    weights = None
    if weighted:
        rng = np.random.default_rng(5)
        weights = rng.uniform(0.25, 1.5, N).astype(np.float32)
        out = rng.random(N) < 0.25
        weights[out] = 0.0
        x[out] = np.inf
    check(x, w, t, weights, dtype, dx, dw, softcap, mean, d_total=0.375, shift=shift, calls=2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_no_row_takes_part(gpu_lib, dtype):
    x, w, t = inputs(70, 64, 90, dtype, 1)
    check(x * np.nan, w, np.full(70, -1), dtype=dtype)
    check(x * np.nan, w, t, np.zeros(70, np.float32), dtype=dtype)
    check(x[:0], w, t[:0], dtype=dtype, max_rows=4)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("want", ["dx", "dw"])
def test_one_gradient(gpu_lib, dtype, want):
    x, w, t = inputs(150, 72, 330, dtype, 2, pad=0.2)
    check(x, w, t, dtype=dtype, want_dx=want == "dx", want_dw=want == "dw")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", [8.0, 60.0, 4000.0])
def test_logits_far_apart(gpu_lib, dtype, size):
    """Logits whose differences leave fp32's exponentials, targets far below the largest."""
    N, D, V = 96, 64, 700
    rng = np.random.default_rng(11)
    w = as_kept(rng.standard_normal((V, D)) * (size / np.sqrt(D)), dtype)
    x = as_kept(rng.standard_normal((N, D)), dtype)
    l = x.astype(np.float64) @ w.T.astype(np.float64)
    t = rng.integers(0, V, N)
    t[:32] = l[:32].argmax(axis=1)  # losses next to zero
    t[32:64] = l[32:64].argmin(axis=1)
    check(x, w, t, dtype=dtype)


def test_infinite_logits_of_others(gpu_lib):
    """A vocabulary entry at minus infinity is one that cannot come: no probability, no
    gradient of the logits, every finite output as without it."""
    N, D, V = 40, 64, 200
    x, w, t = inputs(N, D, V, "fp32", 12)
    x[:, 0] = np.abs(x[:, 0]) + 0.5
    out = np.array([3, 77, 199])
    t[np.isin(t, out)] = 5
    keep = np.setdiff1d(np.arange(V), out)
    w2 = w.copy()
    w2[out] = 0.0
    w2[out, 0] = -np.inf
    dxi, dwi, dti = Dev(x), Dev(w2), Dev(t.astype(np.int32), "int32")
    loss, lse = Dev.out((N,)), Dev.out((N,))
    with TokenLoss(V, D, N, dtype="fp32", backward=False) as h:
        h.forward(N, dxi.ptr, dwi.ptr, dti.ptr, loss=loss.ptr, lse=lse.ptr)
        h.synchronize()
    at = np.searchsorted(keep, t)
    ref = token_loss(x, w[keep], at)
    row, _, _ = tolerances(x, w[keep], ref, "fp32", 0.0, V)
    close(loss.get(), ref["loss"], row, "fp32", "loss")
    close(lse.get(), ref["lse"], row, "fp32", "lse")


def test_a_nan_row_stays_its_own(gpu_lib):
    """A row that takes part and holds a NaN: its loss, lse and dx are NaN, other rows'
    are what they are."""
    N, D, V = 130, 64, 300
    x, w, t = inputs(N, D, V, "bf16", 13)
    x2 = x.copy()
    x2[70, 5] = np.nan
    outs = []
    for v in (x, x2):
        dx_, dw_, dt = Dev(v, "bf16"), Dev(w, "bf16"), Dev(t.astype(np.int32), "int32")
        loss, lse, gx = Dev.out((N,)), Dev.out((N,)), Dev.out((N, D))
        with TokenLoss(V, D, N, mean=False) as h:
            h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, loss=loss.ptr, lse=lse.ptr)
            h.synchronize()
        outs.append((loss.get(), lse.get(), gx.get()))
    others = np.arange(N) != 70
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a[others], b[others])
        assert np.all(np.isnan(b[70]))


@pytest.mark.parametrize("dtype,dw", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32"), ("fp32", "bf16")])
def test_pieces(gpu_lib, dtype, dw, monkeypatch):
    """Rows in several pieces, the last one partly filled or empty of rows that take part."""
    N, D, V = 1100, 72, 600
    monkeypatch.setenv("MXM_XENT_PIECE_BYTES", str(300 * 640 * 2))
    for pad in (0.0, 0.6):
        x, w, t = inputs(N, D, V, dtype, 17, pad=pad)
        check(x, w, t, dtype=dtype, dx_dtype=dtype, dw_dtype=dw, softcap=20.0)


def test_one_handle_many_sizes(gpu_lib):
    """Fewer rows than before on one handle: nothing of the earlier call is left."""
    D, V = 72, 500
    with TokenLoss(V, D, 700, dtype="bf16") as h:
        for N in (700, 1, 333, 64, 2):
            x, w, t = inputs(N, D, V, "bf16", N, pad=0.2)
            check(x, w, t, dtype="bf16", handle=h)


def test_rows_behind_are_left(gpu_lib):
    x, w, t = inputs(100, 64, 128, "bf16", 3)
    dx_, dw_, dt = Dev(x, "bf16"), Dev(w, "bf16"), Dev(t.astype(np.int32), "int32")
    loss, gx = Dev.out((100,)), Dev.out((100, 64))
    with TokenLoss(128, 64, 100) as h:
        h.backward(60, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, loss=loss.ptr)
        h.synchronize()
    assert np.all(loss.get()[60:].view(np.uint32) == 0x5A5A5A5A)
    assert np.all(gx.get()[60:].view(np.uint32) == 0x5A5A5A5A)


def test_refusals(gpu_lib):
    b = Dev(np.zeros(16384, np.float32))
    t = Dev(np.zeros(8, np.int32), "int32")
    o = Dev.out((64,))
    x, w = b.ptr, b.ptr + 4096
    with TokenLoss(16, 8, 8, dtype="fp32", backward=False) as h:
        for call, what in (
                (lambda: h.forward(9, x, w, t.ptr, total=o.ptr), "rows 9 out of range"),
                (lambda: h.forward(8, 0, w, t.ptr, total=o.ptr), "x must be non-NULL"),
                (lambda: h.forward(8, x, 0, t.ptr, total=o.ptr), "weight must be non-NULL"),
                (lambda: h.forward(8, x, w, 0, total=o.ptr), "targets must be non-NULL"),
                (lambda: h.forward(8, x, w, t.ptr), "needs loss, lse or total"),
                (lambda: h.forward(8, x + 2, w, t.ptr, total=o.ptr), "not aligned"),
                (lambda: h.forward(8, x, w, t.ptr, loss=o.ptr, lse=o.ptr + 4), "overlaps"),
                (lambda: h.forward(8, x, w, t.ptr, loss=x), "overlaps"),
                (lambda: h.backward(8, x, w, t.ptr, dx=o.ptr), "MXM_XENT_BACKWARD")):
            with pytest.raises(_lib.MixMoEError, match=what):
                call()
    with TokenLoss(16, 8, 8, dtype="fp32") as h:
        for call, what in (
                (lambda: h.backward(8, x, w, t.ptr), "needs dx or dw"),
                (lambda: h.backward(8, x, w, t.ptr, dx=x), "overlaps"),
                (lambda: h.backward(8, x, w, t.ptr, dw=w), "overlaps"),
                (lambda: h.backward(8, x, w, t.ptr, dx=o.ptr, d_total=float("nan")), "d_total must be finite")):
            with pytest.raises(_lib.MixMoEError, match=what):
                call()
