"""The gradient of capped logits, entry by entry: a table whose row v has a one in the
channel 1 + v, for rows of x that are zero but for channel 0, so that dx holds the logits'
own gradient."""
import numpy as np
import pytest

from mixlab_amd.vocab import TokenLoss
from tests.train_testutil import U32, UBF, Dev, as_kept, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("cap", [1 / 64, 1.0, 30.0, 1024.0])
# logits in blocks of 32, 64 and 128 entries
@pytest.mark.parametrize("N,V", [(33, 61), (2500, 999), (4300, 2001)])
def test_gradient_of_saturated_logits(gpu_lib, N, V, cap, dtype):
    """Logits to twelve caps on both sides: the cap's slope, down to 1.5e-10, keeps its
    digits, of targets and of others."""
    rng = np.random.default_rng(V)
    w = np.zeros((V, V + 1), np.float32)
    w[:, 0] = as_kept(rng.uniform(-12, 12, V) * cap, dtype)
    w[np.arange(V), 1 + np.arange(V)] = 1.0
    x = np.zeros((N, V + 1), np.float32)
    x[:, 0] = rng.choice(np.array([1.0, 0.75, 0.5, -1.0], np.float32), N)
    t = rng.integers(0, V, N).astype(np.int32)
    dx_, dw_, dt, gx = Dev(x, dtype), Dev(w, dtype), Dev(t, "int32"), Dev.out((N, V + 1))
    with TokenLoss(V, V + 1, N, dtype=dtype, softcap=cap, mean=False) as h:
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr)
        h.synchronize()
    z = x[:, :1].astype(np.float64) * w[:, 0]
    l = cap * np.tanh(z / cap)
    p = np.exp(l - l.max(axis=1, keepdims=True))
    whole = p.sum(axis=1, keepdims=True)
    rows = np.arange(N)
    others = p.copy()
    others[rows, t] = 0.0
    dl = p / whole
    dl[rows, t] = -(others.sum(axis=1, keepdims=True) / whole)[:, 0]
    e = np.exp(-2 * np.abs(z) / cap)
    want = dl * 4 * e / (1 + e) ** 2
    # of a share: a capped logit is off by a few roundings of the cap, the row's sum and the
    # exponentials by the steps of V additions; of the slope: an exponential of 2 |z| / cap
    # (an argument of twice that in roundings), a reciprocal and four products
    rel = 16 * U32 * cap + U32 * (16 * np.abs(l).max() + 2 * (V / 64 + 160)) + U32 * (8 * np.abs(z) / cap + 16)
    most = np.abs(dl).max(axis=1, keepdims=True)
    if dtype == "bf16":
        # summands in fp16, to 2^-39 of their block's largest exponential; then bf16
        bound = np.abs(want) * (rel + UBF + UBF / 4) + most * 2.0 ** -39
    else:
        # planes of the row's largest gradient times its row of the table (without the
        # slope: what the least exponent is made of), the slack of four bits, and factors
        # of two of the exponents
        wtop = np.maximum(np.abs(w[:, 0]), 1.0)[None, :]
        scale = np.maximum((np.abs(want) * wtop).max(axis=1, keepdims=True), most * wtop.max())
        bound = np.abs(want) * (rel + 16 * U32) + 2.0 ** -39 * 8 * 16 * scale / wtop
    # (an entry whose share is below 2^-86 of the row's largest may come as zero)
    bound = bound + most * 2.0 ** -86
    close(gx.get()[:, 1:], want, bound, "fp32", "dz")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N", [40, 700])
def test_rows_that_are_not_numbers(gpu_lib, N, dtype):
    """Under a softcap too a row with a NaN has no number for a loss or a gradient, and the
    other rows' results are what they are without it."""
    V, D = 4100, 24
    rng = np.random.default_rng(N)
    w = as_kept(rng.standard_normal((V, D)), dtype)
    x = as_kept(rng.standard_normal((N, D)), dtype)
    t = rng.integers(0, V, N).astype(np.int32)
    bad = np.array([3, N // 2, N - 1])
    x2 = x.copy()
    x2[bad, 5] = np.nan
    outs = []
    for v in (x, x2):
        dx_, dw_, dt = Dev(v, dtype), Dev(w, dtype), Dev(t, "int32")
        loss, lse, gx, one = Dev.out((N,)), Dev.out((N,)), Dev.out((N, D)), Dev.out((N,))
        with TokenLoss(V, D, N, dtype=dtype, softcap=3.0, mean=False) as h:
            h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, loss=loss.ptr, lse=lse.ptr)
            h.forward(N, dx_.ptr, dw_.ptr, dt.ptr, loss=one.ptr)
            h.synchronize()
        outs.append((loss.get(), lse.get(), gx.get(), one.get()))
    others = np.setdiff1d(np.arange(N), bad)
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a[others], b[others])
        assert np.all(np.isnan(b[bad]))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N,V", [(20, 300), (520, 16500)])
def test_logits_far_past_the_cap(gpu_lib, N, V, dtype):
    """Where the exponential of the cap is infinite, or zero: a capped logit is the cap, its
    slope zero, of others and of targets."""
    cap, D = 2.0, 8
    w = np.zeros((V, D), np.float32)
    kinds = np.array([0.0, 100.0, -100.0, 1e30, -1e30, 1.0], np.float32)
    w[:, 0] = as_kept(kinds[np.arange(V) % 6], dtype)
    x = np.zeros((N, D), np.float32)
    x[:, 0] = 1.0
    t = (np.arange(N) % 6).astype(np.int32)
    dx_, dw_, dt = Dev(x, dtype), Dev(w, dtype), Dev(t, "int32")
    gw, loss, one = Dev.out((V, D)), Dev.out((N,)), Dev.out((N,))
    with TokenLoss(V, D, N, dtype=dtype, softcap=cap, mean=False) as h:
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dw=gw.ptr, loss=loss.ptr)
        h.forward(N, dx_.ptr, dw_.ptr, dt.ptr, loss=one.ptr)
        h.synchronize()
    l = cap * np.tanh(w[:, 0].astype(np.float64) / cap)
    p = np.exp(l) / np.exp(l).sum()
    want = np.log(np.exp(l).sum()) - l[t]
    off = U32 * (64 * cap + 2 * (V / 64 + 160))
    for o in (loss, one):
        close(o.get(), want, off, "fp32", "loss")
    slope = 1 - np.tanh(w[:, 0].astype(np.float64) / cap) ** 2
    dw = N * p
    dw[:6] -= np.bincount(t, minlength=6)
    # (zero within what the slope of 50 caps is, e^-100 and so 2^-144)
    bound = (np.abs(dw) * slope + N * p * slope) * (off + (UBF + UBF / 4 if dtype == "bf16" else 16 * U32) + 2 * N * U32)
    close(gw.get()[:, 0], dw * slope, bound + N * 2.0 ** -39 * p.max() * (slope > 1e-30) + 1e-30, "fp32", "dw")
    assert not np.any(gw.get()[:, 1:])
