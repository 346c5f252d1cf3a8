"""The token loss where numbers or sizes reach far: magnitudes of rows and entries,
weights and scales of any sign, pieces with offsets past 32 bits, tables and batches of
more than 2^31 elements."""
import ctypes

import numpy as np
import pytest

from mixlab_amd import _lib
from mixlab_amd.vocab import TokenEmbedding, TokenLoss
from mixlab_amd.workloads import bf16_bits
from oracle.vocab import token_loss
from tests.test_gpu_xent import check, inputs, tolerances
from tests.train_testutil import U32, UBF, Dev, as_kept, close, from_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ex", [-90, -30, 40, 90])
def test_magnitudes_of_the_operands(gpu_lib, dtype, ex):
    """x times a power of two and the table divided by it: the logits stay."""
    x, w, t = inputs(150, 72, 330, dtype, 21, pad=0.1)
    check(np.ldexp(x, ex).astype(np.float32), np.ldexp(w, -ex).astype(np.float32), t, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_and_entries_of_unlike_magnitude(gpu_lib, dtype):
    rng = np.random.default_rng(3)
    x, w, t = inputs(150, 72, 330, dtype, 22)
    x = np.ldexp(x, rng.integers(-40, 1, (150, 1))).astype(np.float32)
    w = np.ldexp(w, rng.integers(-40, 1, (330, 1))).astype(np.float32)
    x[5] = 0.0
    w[9] = 0.0
    check(x, w, t, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("which", ["some", "most", "all"])
def test_entries_of_zeros(gpu_lib, dtype, which):
    """Rows of the table that hold zeros, or next to nothing: their gradient is as any."""
    x, w, t = inputs(150, 72, 330, dtype, 25)
    out = {"some": [5, 9, 200], "most": np.arange(300), "all": np.arange(330)}[which]
    w[out] = 0.0
    t[3] = 5
    check(x, w, t, dtype=dtype, softcap=20.0 if which == "most" else 0.0)
    w[out] = as_kept(np.random.default_rng(1).standard_normal((len(out), 72)) * 1e-9, dtype)
    check(x, w, t, dtype=dtype)


@pytest.mark.parametrize("dtype,lowest", [("bf16", -3.38e38), ("fp32", -3.38e38), ("fp32", -np.inf)])
def test_masked_entries(gpu_lib, dtype, lowest, monkeypatch):
    """Entries that a first channel of the type's lowest value, or less, keeps from coming
    (x's is above zero): every other result is as without them, their gradient is zero."""
    N, D, V = 700, 72, 330
    x, w, t = inputs(N, D, V, dtype, 26, pad=0.2)
    x[:, 0] = np.abs(x[:, 0]) + 0.5
    x = as_kept(x, dtype)
    out = np.array([3, 77, 299])
    t[np.isin(t, out)] = 5
    w[out, 0] = as_kept(np.array([lowest]), dtype)
    keep = np.setdiff1d(np.arange(V), out)
    took = (t >= 0) & (t < V)
    at = np.where(took, np.searchsorted(keep, np.clip(t, 0, V - 1)), -1)
    clean = np.where(took[:, None], x, 0.0)
    ref = token_loss(clean, w[keep], at)
    row, bx, bw = tolerances(clean[took], w[keep], ref, dtype, 0.0, V)
    for piece in (None, 1):  # of rows: one, or several
        if piece:
            monkeypatch.setenv("MXM_XENT_PIECE_BYTES", str(piece))
        dx_, dw_, dt = Dev(x, dtype), Dev(w, dtype), Dev(t.astype(np.int32), "int32")
        loss, lse, gx, gw = Dev.out((N,)), Dev.out((N,)), Dev.out((N, D)), Dev.out((V, D))
        with TokenLoss(V, D, N, dtype=dtype) as h:
            h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr, loss=loss.ptr, lse=lse.ptr)
            h.synchronize()
        close(loss.get()[took], ref["loss"][took], row, "fp32", "loss")
        close(lse.get()[took], ref["lse"][took], row, "fp32", "lse")
        close(gx.get()[took], ref["dx"][took], bx, "fp32", "dx")
        close(gw.get()[keep], ref["dw"], bw, "fp32", "dw")
        assert not np.any(gw.get()[out])


@pytest.mark.parametrize("cap", [4.0, 1.0])
@pytest.mark.parametrize("dtype,lowest", [("bf16", -3.38e38), ("fp32", -3.38e38), ("fp32", -np.inf)])
def test_masked_entries_under_a_softcap(gpu_lib, dtype, lowest, cap):
    """Their logit is -softcap, as the formula has it, with a slope of zero."""
    N, D, V = 300, 72, 330
    x, w, t = inputs(N, D, V, dtype, 28)
    x[:, 0] = np.abs(x[:, 0]) + 0.5
    x = as_kept(x, dtype)
    out = np.array([3, 77, 78, 299])
    t[np.isin(t, out)] = 5
    keep = np.setdiff1d(np.arange(V), out)
    part = token_loss(x, w[keep], np.searchsorted(keep, t), softcap=cap)
    row, bx, bw = tolerances(x, w[keep], part, dtype, cap, V)
    w[out, 0] = -1e6  # (of a tanh of -1 too)
    ref = token_loss(x, w, t, softcap=cap)
    w[out, 0] = as_kept(np.array([lowest]), dtype)
    dx_, dw_, dt = Dev(x, dtype), Dev(w, dtype), Dev(t.astype(np.int32), "int32")
    loss, lse, gx, gw = Dev.out((N,)), Dev.out((N,)), Dev.out((N, D)), Dev.out((V, D))
    with TokenLoss(V, D, N, dtype=dtype, softcap=cap) as h:
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr, loss=loss.ptr, lse=lse.ptr)
        h.synchronize()
    assert cap > 1.0 or np.all(ref["lse"] - part["lse"] > row)  # (without their share lse is off by more)
    close(loss.get(), ref["loss"], row, "fp32", "loss")
    close(lse.get(), ref["lse"], row, "fp32", "lse")
    close(gx.get(), ref["dx"], bx, "fp32", "dx")
    close(gw.get()[keep], ref["dw"][keep], bw, "fp32", "dw")
    assert not np.any(gw.get()[out])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("cap", [1 / 64, 0.5, 1024.0])
def test_caps(gpu_lib, dtype, cap):
    x, w, t = inputs(150, 72, 330, dtype, 29, pad=0.1)
    check(x, w, t, dtype=dtype, softcap=cap)


@pytest.mark.parametrize("dx,dw", [(True, True), (True, False), (False, True)])
def test_pieces_of_unlike_magnitude(gpu_lib, dx, dw, monkeypatch):
    """Under fp32, pieces whose gradients reach rows of the table of ever larger or ever
    smaller magnitude: each piece moves the small rows' common exponent, or leaves it."""
    N, D, V = 1100, 72, 400
    rng = np.random.default_rng(2)
    ex = np.sort(rng.integers(-24, 1, V))
    for down in (False, True):
        monkeypatch.setenv("MXM_XENT_PIECE_BYTES", "1")
        x, w, t = inputs(N, D, V, "fp32", 27)
        w[:, 0] = 1.0
        w = np.ldexp(w, ex[:, None]).astype(np.float32)
        w[7] = 0.0
        # channel 0 keeps the rows from coming that are above 2^-at or so
        at = 22 - 5 * (np.arange(N) // 256)
        at = at[::-1] if down else at
        x[:, 0] = -np.ldexp(1.0, at)
        t = np.array([rng.integers(0, np.searchsorted(ex, 2 - a)) for a in at])
        check(x, w, t, dtype="fp32", want_dx=dx, want_dw=dw)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V,pad,weighted,shift", [
    (1, 2048, 3000, 0.0, False, 0), (1, 64, 500, 1.0, False, 0), (2, 72, 40000, 0.0, True, 0),
    (17, 136, 700, 0.4, True, 0), (32, 8, 130, 0.3, False, 0), (32, 520, 1000, 0.0, False, 8),
    (4, 40, 33000, 0.0, False, 0), (5, 40, 33001, 0.2, False, 0), (16, 24, 40000, 0.0, True, 0),
    (31, 100, 400, 0.2, True, 0), (33, 136, 700, 0.4, True, 0), (20, 64, 128, 0.5, False, 1)])
def test_few_rows(gpu_lib, N, D, V, pad, weighted, shift, dtype):
    """Up to the few rows that a forward reads in place, in and out of order, and past them."""
    x, w, t = inputs(N, D, V, dtype, 31 * N + V, pad=pad)
    weights = None
    if weighted:
        weights = np.random.default_rng(N).uniform(0.5, 1.5, N).astype(np.float32)
        weights[1::3] = 0.0
        x[1::3] = np.nan
    check(x, w, t, weights, dtype=dtype, softcap=25.0 if N % 2 else 0.0, shift=shift, calls=2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V,weighted,pad", [
    (40, 16384, 70, False, 0.0), (6, 16383, 130, True, 0.0), (300, 2056, 1, False, 0.2),
    (4096, 40, 90, True, 0.3), (4097, 40, 90, True, 0.3), (9001, 24, 65, True, 0.6)])
def test_extreme_sizes(gpu_lib, N, D, V, weighted, pad, dtype):
    """The widest rows, a table of one entry, batches around the counts' own launch."""
    x, w, t = inputs(N, D, V, dtype, N + D, pad=pad)
    weights = np.random.default_rng(V).uniform(0.5, 1.5, N).astype(np.float32) if weighted else None
    check(x, w, t, weights, dtype=dtype, calls=2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_elements_of_unlike_magnitude(gpu_lib, dtype):
    """Within a row of x and of the table: below the planes' reach an element counts as
    far as its share of the row's largest."""
    rng = np.random.default_rng(4)
    x, w, t = inputs(90, 136, 200, dtype, 23)
    x = np.ldexp(x, rng.integers(-30, 1, x.shape)).astype(np.float32)
    w = np.ldexp(w, rng.integers(-30, 1, w.shape)).astype(np.float32)
    check(as_kept(x, dtype), as_kept(w, dtype), t, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d_total", [0.0, -3.0, 65536.0, 2.0 ** -40, 2.0 ** 60])
def test_scales_of_the_gradient(gpu_lib, dtype, d_total):
    rng = np.random.default_rng(5)
    x, w, t = inputs(120, 64, 200, dtype, 24, pad=0.2)
    weights = rng.uniform(-1.0, 2.0, 120).astype(np.float32)  # some below zero
    weights[::9] = 0.0
    check(x, w, t, weights, dtype=dtype, d_total=d_total, mean=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_that_are_not_finite_stay_their_own(gpu_lib, dtype):
    """A NaN or an infinity in a row that takes part leaves the others' results as they
    are, in whatever tile or group of rows they lie."""
    N, D, V = 700, 72, 300
    x, w, t = inputs(N, D, V, dtype, 13)
    x2 = x.copy()
    bad = np.array([3, 70, 130, 611])
    x2[bad, 5] = [np.nan, np.inf, -np.inf, np.nan]
    outs = []
    for v in (x, x2):
        dx_, dw_, dt = Dev(v, dtype), Dev(w, dtype), Dev(t.astype(np.int32), "int32")
        loss, lse, gx = Dev.out((N,)), Dev.out((N,)), Dev.out((N, D))
        with TokenLoss(V, D, N, dtype=dtype, mean=False) as h:
            h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, loss=loss.ptr, lse=lse.ptr)
            h.synchronize()
        outs.append((loss.get(), lse.get(), gx.get()))
    others = np.setdiff1d(np.arange(N), bad)
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a[others], b[others])
        assert not np.any(np.isfinite(b[bad[[0, 3]]]))


def test_weights_that_cancel_leave_no_mean(gpu_lib):
    """Weights that sum to zero: the mean divides by it, as its formula does."""
    x, w, t = inputs(4, 64, 90, "bf16", 2)
    rw = Dev(np.array([1, -1, 2, -2], np.float32))
    dx_, dw_, dt = Dev(x, "bf16"), Dev(w, "bf16"), Dev(t.astype(np.int32), "int32")
    loss, total, gx = Dev.out((4,)), Dev.out((1,)), Dev.out((4, 64))
    with TokenLoss(90, 64, 4) as h:
        h.backward(4, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, row_weights=rw.ptr, loss=loss.ptr, total=total.ptr)
        h.synchronize()
    ref = token_loss(x, w, t)
    row, _, _ = tolerances(x, w, ref, "bf16", 0.0, 90)
    close(loss.get(), ref["loss"], row, "fp32", "loss")
    assert not np.isfinite(total.get()[0]) and not np.any(np.isfinite(gx.get()))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N,V,piece", [(9000, 262_145, 64 << 30), (300, 4_194_304, 0)])
def test_pieces_past_32_bit_offsets(gpu_lib, dtype, N, V, piece, monkeypatch):
    """Logits of over 2^31 elements in one piece, and pieces of the longest table.  The
    rows are four, over and over, which the restatement gives as often as they occur."""
    if dtype == "fp32" and N > 300:
        N = 8300  # (8 bytes of workspace each)
    D, k = 8, 4
    monkeypatch.setenv("MXM_XENT_PIECE_BYTES", str(piece or 1))
    x, w, t = inputs(k, D, V, dtype, 5)
    t[0], t[1] = V - 1, 0
    which = np.random.default_rng(1).integers(0, k, N)
    count = np.bincount(which, minlength=k).astype(np.float64)
    ref = token_loss(x, w, t, count, mean=False)
    row, bx, bw = tolerances(x, w, ref, dtype, 0.0, V)
    bw = bw + 2 * (3 if dtype == "fp32" else 1) * N * U32 * (np.abs(ref["dz"]).T @ np.abs(x))
    bx = bx / count[:, None]
    dx_, dw_, dt = Dev(x[which], dtype), Dev(w, dtype), Dev(t[which].astype(np.int32), "int32")
    loss, lse, total = Dev.out((N,)), Dev.out((N,)), Dev.out((1,))
    gx, gw = Dev.out((N, D)), Dev.out((V, D))
    with TokenLoss(V, D, N, dtype=dtype, mean=False) as h:
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr, loss=loss.ptr, lse=lse.ptr, total=total.ptr)
        h.synchronize()
    close(loss.get(), ref["loss"][which], row[which], "fp32", "loss")
    close(lse.get(), ref["lse"][which], row[which], "fp32", "lse")
    close(total.get(), ref["total"], (count * (row + 2 * U32 * ref["loss"])).sum(), "fp32", "total")
    close(gx.get(), (ref["dx"] / count[:, None])[which], bx[which], "fp32", "dx")
    close(gw.get(), ref["dw"], bw, "fp32", "dw")


def _zeros(nbytes):
    b = _lib.DeviceBuffer(nbytes)
    assert _lib.load().hipMemset(ctypes.c_void_p(b.value), 0, ctypes.c_size_t(nbytes)) == 0
    return b


def _put(buf, at, a):
    a = np.ascontiguousarray(a)
    _lib.check(_lib.load().mxm_memcpy_h2d(buf.value + at, a.ctypes.data, a.nbytes), "h2d")


def _get(buf, at, shape):
    out = np.empty(shape, np.uint16)
    _lib.check(_lib.load().mxm_memcpy_d2h(out.ctypes.data, buf.value + at, out.nbytes), "d2h")
    return from_bits(out)


def test_table_past_2_31_elements(gpu_lib):
    """The longest table at a width of 520 (2.2e9 elements), zero but for its last rows:
    lookups, the loss with both gradients, and the embedding's gradient on top."""
    V, D, N, k = 4_194_304, 520, 5, 200
    rng = np.random.default_rng(0)
    far = as_kept(rng.standard_normal((k, D)) * 0.1, "bf16")
    x = as_kept(rng.standard_normal((N, D)), "bf16")
    t = np.array([V - 1, V - k, V - 7, V - 100, V - 2], np.int32)
    table, grad = _zeros(V * D * 2), _zeros(V * D * 2)
    _put(table, (V - k) * D * 2, bf16_bits(far))
    dt, out = Dev(t, "int32"), Dev.out((N, D), "bf16")
    dx_, loss, gx = Dev(x, "bf16"), Dev.out((N,)), Dev.out((N, D))
    tail = far.astype(np.float64)
    with TokenEmbedding(V, D, N, "bf16", "bf16", "fp32", "bf16") as e, \
            TokenLoss(V, D, N, dw_dtype="bf16", share=e) as h:
        e.forward(N, dt.ptr, table.value, out.ptr)
        h.backward(N, dx_.ptr, table.value, dt.ptr, dx=gx.ptr, dw=grad.value, loss=loss.ptr)
        h.synchronize()
        np.testing.assert_array_equal(out.get(), far[t - (V - k)])
        near, end = _get(grad, 0, (64, D)), _get(grad, (V - k) * D * 2, (k, D))
        # the rows of zeros have the logit 0: one of them stands for all
        x64 = x.astype(np.float64)
        l = x64 @ tail.T
        size = np.abs(x64) @ np.abs(tail).T
        lse = np.log(np.exp(l).sum(axis=1) + (V - k))
        at = t - (V - k)
        err = (2 * (D + 8) + 4) * U32 * size.max() + U32 * (8 * np.abs(l).max() + 2 * (V / 64 + 160))
        close(loss.get(), lse - l[np.arange(N), at], 2 * err, "fp32", "loss")
        p = np.exp(l - lse[:, None]) / N
        edz = p * (2 * err + 1.25 * UBF)
        p[np.arange(N), at] -= 1 / N
        edz[np.arange(N), at] = (np.abs(p) * (2 * err + 1.25 * UBF))[np.arange(N), at]
        sums = (V + 64) * 2 * U32
        close(gx.get(), p @ tail, edz @ np.abs(tail) + sums * (np.abs(p) + edz) @ np.abs(tail), "fp32", "dx")
        close(end, p.T @ x64, edz.T @ np.abs(x64) + 2 * (N + 64) * U32 * np.abs(p).T @ np.abs(x64), "bf16", "dw")
        p0 = np.exp(-lse) / N
        want = np.broadcast_to(p0 @ x64, near.shape)
        # (fp16 summands of a block keep 2^-39 of its largest at least: of equal ones, all)
        close(near, want, (2 * err + 1.25 * UBF + 2 * (N + 64) * U32) * (p0 @ np.abs(x64)), "bf16", "dw of zero rows")
        before = end
        e.backward(N, dt.ptr, gx.ptr, grad.value, accumulate=True)
        e.synchronize()
        after = _get(grad, (V - k) * D * 2, (k, D))
        g = gx.get().astype(np.float64)
        want = before.astype(np.float64)
        want[at] += g
        close(after, want, 3 * U32 * (np.abs(before) + np.abs(want)), "bf16", "d_table")
        np.testing.assert_array_equal(_get(grad, 0, (64, D)), near)
        e.backward(N, dt.ptr, gx.ptr, grad.value)
        e.synchronize()
        assert not np.any(_get(grad, 0, (64, D)))
        want = np.zeros((k, D))
        want[at] = g
        close(_get(grad, (V - k) * D * 2, (k, D)), want, 0 * want, "bf16", "d_table")


@pytest.mark.parametrize("taking", ["last", "all"])
def test_rows_past_2_31_elements(gpu_lib, taking):
    """4.2 million rows of 520, zero but for the last: only those take part, or all."""
    N, D, V, k = 4_200_000, 520, 130, 150
    rng = np.random.default_rng(2)
    w = as_kept(rng.standard_normal((V, D)) * 0.1, "bf16")
    far = as_kept(rng.standard_normal((k, D)), "bf16")
    t = rng.integers(0, V, N).astype(np.int32)
    if taking == "last":
        t[:N - k] = -1
    x, gx = _zeros(N * D * 2), _zeros(N * D * 2)
    _put(x, (N - k) * D * 2, bf16_bits(far))
    dw_, dt, loss, gw = Dev(w, "bf16"), Dev(t, "int32"), Dev.out((N,)), Dev.out((V, D))
    with TokenLoss(V, D, N, dx_dtype="bf16", mean=False) as h:
        h.backward(N, x.value, dw_.ptr, dt.ptr, dx=gx.value, dw=gw.ptr, loss=loss.ptr)
        h.synchronize()
    ref = token_loss(far, w, t[N - k:], mean=False)
    row, bx, bw = tolerances(far, w, ref, "bf16", 0.0, V)
    got = loss.get()
    close(got[N - k:], ref["loss"], row, "fp32", "loss")
    close(_get(gx, (N - k) * D * 2, (k, D)), ref["dx"], bx, "bf16", "dx")
    close(gw.get(), ref["dw"], bw, "fp32", "dw")  # (rows of zeros add none)
    near = _get(gx, 0, (64, D))
    if taking == "last":
        assert not np.any(got[:N - k]) and not np.any(near)
    else:
        zero = token_loss(np.zeros((64, D)), w, t[:64], mean=False)
        _, b, _ = tolerances(np.zeros((64, D)), w, zero, "bf16", 0.0, V)
        close(got[:N - k], np.log(V), 2 * U32 * (2 * (V / 64 + 160)), "fp32", "loss")
        close(near, zero["dx"], b, "bf16", "dx")
