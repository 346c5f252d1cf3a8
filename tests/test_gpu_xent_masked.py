"""The token loss where whole blocks of the vocabulary are masked: an entry that a first
channel far below zero keeps from coming has no share in any result, wherever it lies."""
import numpy as np
import pytest

from mixlab_amd.vocab import TokenLoss
from oracle.vocab import token_loss
from tests.test_gpu_xent import inputs, tolerances
from tests.train_testutil import Dev, as_kept, close

pytestmark = pytest.mark.gpu

LOWEST = {"bf16": -3.38e38, "fp32": -3.4e38}


def masked(which, V):
    if which == "tail":          # a table padded to whole tiles
        return np.arange(V - V // 5, V)
    if which == "runs":          # whole blocks of 32, 64 and 128 entries, and one across them
        return np.concatenate([np.arange(a, min(a + n, V)) for a, n in ((0, 128), (160, 32), (256, 64), (400, 99))])
    return np.setdiff1d(np.arange(V), [V // 2])  # all but one


def run(N, D, V, dtype, lowest, out, seed, pad=0.0, softcap=0.0):
    """The results, and those of the table without the masked entries; no target is one."""
    x, w, t = inputs(N, D, V, dtype, seed, pad=pad)
    x[:, 0] = np.abs(x[:, 0]) + 0.5
    x = as_kept(x, dtype)
    keep = np.setdiff1d(np.arange(V), out)
    took = (t >= 0) & (t < V)
    t[took & np.isin(t, out)] = keep[0]
    # rows whose target is the only entry of its block that comes
    for a in (0, 160, 256):
        if np.isin(a, out) and V > 400:
            keep = np.union1d(keep, [a + 7])
            t[np.flatnonzero(took)[a % 7::9]] = a + 7
    out = np.setdiff1d(out, keep)
    w[out, 0] = as_kept(np.array([lowest]), dtype)
    at = np.where(took, np.searchsorted(keep, np.clip(t, 0, V - 1)), -1)
    clean = np.where(took[:, None], x, 0.0)
    ref = token_loss(clean, w[keep], at, softcap=softcap)
    row, bx, bw = tolerances(clean[took], w[keep], ref, dtype, softcap, V)
    dx_, dw_, dt = Dev(x, dtype), Dev(w, dtype), Dev(t.astype(np.int32), "int32")
    gx, gw = Dev.out((N, D)), Dev.out((V, D))
    both = [[Dev.out((N,)), Dev.out((N,)), Dev.out((1,))] for _ in range(2)]
    with TokenLoss(V, D, N, dtype=dtype) as h:
        a, b = both
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr, loss=a[0].ptr, lse=a[1].ptr, total=a[2].ptr)
        h.forward(N, dx_.ptr, dw_.ptr, dt.ptr, loss=b[0].ptr, lse=b[1].ptr, total=b[2].ptr)
        h.synchronize()
    for loss, lse, total in both:
        close(loss.get()[took], ref["loss"][took], row, "fp32", "loss")
        close(lse.get()[took], ref["lse"][took], row, "fp32", "lse")
        close(total.get(), ref["total"], row.max() + 2.0 ** -23 * np.abs(ref["loss"]).max(), "fp32", "total")
    close(gx.get()[took], ref["dx"][took], bx, "fp32", "dx")
    assert not np.any(gx.get()[~took])
    got = gw.get()
    close(got[keep], ref["dw"], bw, "fp32", "dw")
    assert not np.any(got[out])


# few rows and many: blocks of 32, 64 and 128 entries
SMALL = [((n, 72, 530), lowest) for n in (20, 150) for lowest in ("type's", -2.5e38, -1e30, -1e10, -1e9, -3e7, -1e6)]
LARGE = [(s, lowest) for s in ((700, 40, 4100), (520, 24, 16500)) for lowest in ("type's", -1e9)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("which", ["tail", "runs", "all but one"])
@pytest.mark.parametrize("size,lowest", SMALL + LARGE)
def test_masked_blocks(gpu_lib, size, which, lowest, dtype):
    N, D, V = size
    lowest = LOWEST[dtype] if lowest == "type's" else lowest
    run(N, D, V, dtype, lowest, masked(which, V), N + V, pad=0.1)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_logits_far_from_zero(gpu_lib, dtype):
    """Rows whose logits are all of some magnitude, with distances that it keeps: one entry
    in 97 has a logit of 2^k, 2^k (1 + 1/128), ..., the others none that matters."""
    N, V, D = 40, 530, 8
    for k in (21, 22, 23, 26, 30, 60, 100):
        x = np.zeros((N, D), np.float32)
        x[:, 0], x[:, 1] = 2.0 ** (k // 2), np.arange(N) % 3
        w = np.zeros((V, D), np.float32)
        at = np.arange(5, V, 97)
        w[at, 0] = np.ldexp(1.0 + np.arange(len(at)) / 128, k - k // 2)
        t = np.full(N, at[-1], np.int32)
        t[::2] = at[0]  # (its loss is the logits' distance)
        ref = token_loss(x, w, t, mean=False)
        dx_, dw_, dt, loss, lse = Dev(x, dtype), Dev(w, dtype), Dev(t, "int32"), Dev.out((N,)), Dev.out((N,))
        gx = Dev.out((N, D))
        with TokenLoss(V, D, N, dtype=dtype, mean=False) as h:
            h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, loss=loss.ptr, lse=lse.ptr)
            h.synchronize()
        # the logits are exact; a block's reference is off by half a step of theirs, and so
        # is the target's place to it
        step = 4 * 2.0 ** -24 * 2.0 ** (k + 1)
        close(lse.get(), ref["lse"], step, "fp32", f"lse at 2^{k}")
        close(loss.get(), ref["loss"], 2 * step, "fp32", f"loss at 2^{k}")
        close(gx.get()[::2], ref["dx"][::2], 2.0 ** -7 * np.abs(ref["dx"][::2]), "fp32", f"dx at 2^{k}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [1, 40, 300])
def test_only_the_target_comes(gpu_lib, V, dtype):
    """Loss and gradients are zero, also where the target's own logit is far below zero."""
    D, N = 16, 9
    for own in (0.5, -1e4, -1e30):
        x = np.ones((N, D), np.float32)
        w = np.zeros((V, D), np.float32)
        w[:, 0] = LOWEST[dtype] if own > -1e30 else -np.inf
        w[V // 2, 0] = own
        w = as_kept(w, dtype)
        if dtype == "bf16" and own == -1e30:
            x[:, 1:] = 0.0  # (dx of a bf16 table with infinities is not a number)
        dx_, dw_, dt = Dev(x, dtype), Dev(w, dtype), Dev(np.full(N, V // 2, np.int32), "int32")
        gx, gw, loss, lse = Dev.out((N, D)), Dev.out((V, D)), Dev.out((N,)), Dev.out((N,))
        with TokenLoss(V, D, N, dtype=dtype) as h:
            h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr, loss=loss.ptr, lse=lse.ptr)
            h.synchronize()
        assert not np.any(loss.get()) and not np.any(gw.get())
        close(lse.get(), np.full(N, float(w[V // 2, 0])), 0.0, "fp32", "lse")
        if dtype == "fp32" or own != -1e30:
            assert not np.any(gx.get())
