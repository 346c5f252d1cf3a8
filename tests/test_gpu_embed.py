"""The token embedding on the device against its 64-bit restatement: tokens outside
the table, runs of one token over many chunks, odd widths, alignments and types,
addition to a tied gradient."""
from __future__ import annotations

import numpy as np
import pytest

from mixlab_amd import _lib
from mixlab_amd.vocab import TokenEmbedding
from oracle.vocab import embed_backward, embed_forward
from train_testutil import U32, Dev, as_kept, close

pytestmark = pytest.mark.gpu


def tokens_of(kind, rng, N, V):
    if kind == "uniform":
        t = rng.integers(0, V, N)
    elif kind == "one":          # one token only
        t = np.full(N, V // 2)
    elif kind == "outside":      # none inside
        t = np.where(rng.random(N) < 0.5, -1, V + rng.integers(0, 3, N))
    elif kind == "extremes":
        t = rng.choice(np.array([-2 ** 31, -1, 0, V - 1, V, 2 ** 31 - 1]), N)
    elif kind == "half":         # every other place or so of one token
        t = np.where(rng.random(N) < 0.5, V // 3, rng.integers(0, V, N))
    elif kind == "blocks":       # tokens that occur 64, 128 or 256 times, or one less or more
        n = rng.choice(np.array([1, 63, 64, 65, 127, 128, 129, 256, 257]), N)
        t = rng.permutation(np.repeat(np.arange(N), n)[:N] % V)
    else:                        # skewed, some of them padding
        t = np.minimum((V ** rng.random(N)).astype(np.int64) - 1, V - 1)
        t[rng.random(N) < 0.2] = -1
    return t.astype(np.int32)


@pytest.mark.parametrize("N,D,V,table,out,shift,kind", [
    (1, 64, 100, "fp32", "fp32", 0, "uniform"),
    (8, 1024, 513, "bf16", "fp32", 0, "skewed"),
    (1, 1, 1, "fp32", "bf16", 0, "uniform"),
    (33, 85, 77, "fp32", "bf16", 0, "extremes"),
    (257, 2056, 31, "bf16", "bf16", 0, "skewed"),
    (100, 544, 300, "bf16", "fp32", 1, "extremes"),
    (64, 136, 40, "fp32", "fp32", 3, "outside"),
    (3000, 8, 5000, "bf16", "bf16", 0, "uniform"),
    (130, 100, 90, "bf16", "bf16", 0, "skewed"),
    (130, 72, 90, "bf16", "bf16", 4, "skewed"),
    (20000, 300, 50, "bf16", "bf16", 2, "skewed"),
    (7, 16384, 30, "bf16", "fp32", 0, "extremes"),
    (9, 16383, 30, "fp32", "bf16", 0, "skewed"),
])
def test_forward(gpu_lib, N, D, V, table, out, shift, kind):
    rng = np.random.default_rng(N + D)
    t = tokens_of(kind, rng, N, V)
    w = as_kept(rng.standard_normal((V, D)), table)
    dt, dw = Dev(t, "int32"), Dev(w, table, shift)
    do = Dev.out((N, D), out, shift)
    with TokenEmbedding(V, D, N, table_dtype=table, out_dtype=out, scale=2.75, backward=False) as e:
        e.forward(N, dt.ptr, dw.ptr, do.ptr)
        e.synchronize()
    want = embed_forward(t, w, 2.75)
    close(do.get(), want, U32 * np.abs(want), out, "out")


@pytest.mark.parametrize("N,D,V,grad,dtable,shift,kind,add", [
    (0, 64, 50, "fp32", "fp32", 0, "uniform", False),
    (0, 64, 50, "fp32", "fp32", 0, "uniform", True),
    (1, 64, 50, "fp32", "fp32", 0, "uniform", False),
    (1024, 64, 1024, "fp32", "fp32", 0, "skewed", False),
    (1000, 544, 300, "bf16", "fp32", 0, "skewed", True),
    (777, 85, 33, "fp32", "bf16", 0, "uniform", False),
    (500, 24, 700, "bf16", "bf16", 1, "extremes", False),
    (4097, 72, 3, "fp32", "fp32", 0, "one", True),
    (4096, 2056, 5, "bf16", "fp32", 0, "one", False),
    (300, 40, 90, "fp32", "fp32", 0, "outside", False),
    (300, 40, 90, "fp32", "bf16", 0, "outside", True),
    (40001, 16, 9000, "fp32", "fp32", 0, "skewed", False),
    (33000, 9, 1, "bf16", "fp32", 0, "one", False),
    (65, 8, 20000, "fp32", "fp32", 0, "uniform", False),
    (700, 100, 90, "bf16", "bf16", 0, "skewed", True),
    (1024, 64, 1024, "fp32", "fp32", 0, "one", False),
    (2048, 32, 1, "bf16", "fp32", 0, "one", True),
    (2048, 32, 1000, "fp32", "bf16", 0, "skewed", False),
    (2047, 24, 300, "bf16", "bf16", 1, "extremes", True),
    (9, 1024, 5000, "fp32", "fp32", 0, "extremes", True),
    (8, 2048, 20000, "fp32", "bf16", 0, "uniform", False),
    (2049, 32, 700, "fp32", "fp32", 0, "skewed", True),
    (70, 16384, 9, "bf16", "fp32", 0, "skewed", True),
    (50, 16383, 7, "fp32", "bf16", 0, "extremes", False),
    (40000, 8, 700000, "fp32", "fp32", 0, "skewed", True),
    (5000, 72, 40, "fp32", "fp32", 0, "half", False),
    (20000, 260, 3000, "bf16", "fp32", 0, "half", True),
    (50000, 40, 2000, "fp32", "bf16", 0, "half", False),
    (9000, 24, 5000, "fp32", "fp32", 0, "blocks", False),
    (36000, 24, 5000, "bf16", "bf16", 0, "blocks", True),
    (1900, 32, 300, "fp32", "fp32", 0, "blocks", False),
    (2000, 32, 200, "fp32", "fp32", 0, "half", True),
    (700, 72, 90, "bf16", "bf16", 4, "skewed", False),
    (700, 72, 90, "bf16", "fp32", 2, "skewed", False),
])
def test_backward(gpu_lib, N, D, V, grad, dtable, shift, kind, add):
    rng = np.random.default_rng(N + 3 * D)
    t = tokens_of(kind, rng, N, V)
    dy = rng.standard_normal((N, D))
    dy[(t < 0) | (t >= V)] = np.nan  # never read
    dy = as_kept(dy, grad)
    before = as_kept(rng.standard_normal((V, D)), dtable)
    before[V // 3] = np.nan if add and not np.any(t == V // 3) else before[V // 3]  # left as it was
    dt, dd = Dev(t, "int32"), Dev(dy, grad, shift)
    dw = Dev(before, dtable, shift)
    with TokenEmbedding(V, D, N, grad_dtype=grad, table_grad_dtype=dtable, scale=-0.625) as e:
        e.backward(N, dt.ptr, dd.ptr, dw.ptr, accumulate=add)
        e.synchronize()
        got = dw.get()
        if not add:  # equal inputs, equal bits
            e.backward(N, dt.ptr, dd.ptr, dw.ptr)
            e.synchronize()
            np.testing.assert_array_equal(dw.get(), got)
    want = embed_backward(t, dy, V, -0.625, before if add else None)
    # a sum of m terms in some order: m - 1 roundings of partial sums, one of the
    # scaling, one of the addition to what was there
    inside = (t >= 0) & (t < V)
    count = np.bincount(t[inside], minlength=V)[:, None]
    mass = embed_backward(t, np.abs(dy), V, 0.625)
    bound = (count + 2) * U32 * (mass + (np.abs(before) if add else 0))
    touched = count[:, 0] > 0
    close(got[touched], want[touched], bound[touched], dtable, "d_table")
    np.testing.assert_array_equal(got[~touched], before[~touched] if add else 0.0)


def test_refusals(gpu_lib):
    buf = Dev(np.zeros(4096, np.float32))
    t = Dev(np.zeros(8, np.int32), "int32")
    with TokenEmbedding(16, 8, 8, backward=False) as e:
        for call, what in (
                (lambda: e.forward(9, t.ptr, buf.ptr, buf.ptr + 8192), "rows 9 out of range"),
                (lambda: e.forward(-1, t.ptr, buf.ptr, buf.ptr + 8192), "rows -1 out of range"),
                (lambda: e.forward(8, 0, buf.ptr, buf.ptr + 8192), "tokens must be non-NULL"),
                (lambda: e.forward(8, t.ptr, 0, buf.ptr + 8192), "table must be non-NULL"),
                (lambda: e.forward(8, t.ptr, buf.ptr, 0), "out must be non-NULL"),
                (lambda: e.forward(8, t.ptr, buf.ptr + 2, buf.ptr + 8192), "not aligned"),
                (lambda: e.forward(8, t.ptr, buf.ptr, buf.ptr + 16 * 8 * 4 - 4), "overlaps"),
                (lambda: e.backward(8, t.ptr, buf.ptr, buf.ptr + 8192), "MXM_EMBED_BACKWARD")):
            with pytest.raises(_lib.MixMoEError, match=what):
                call()
        e.forward(0, 0, 0, 0)
    with TokenEmbedding(16, 8, 8) as e:
        for call, what in (
                (lambda: e.backward(8, t.ptr, buf.ptr, 0), "d_table must be non-NULL"),
                (lambda: e.backward(8, t.ptr, 0, buf.ptr), "d_out must be non-NULL"),
                (lambda: e.backward(8, t.ptr, buf.ptr, buf.ptr), "overlaps")):
            with pytest.raises(_lib.MixMoEError, match=what):
                call()
