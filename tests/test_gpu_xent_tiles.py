"""The token loss in every shape of tiles that its rules choose between, against 64 bits:
logits of few rows, of middling and of large ones, alone and with gradients, with and
without a softcap; products for dx and dw in each of their shapes, whole and split along
their sums.  The sizes are such that 256 compute units take the shapes named."""
import numpy as np
import pytest

from mixlab_amd.vocab import TokenLoss
from oracle.vocab import token_loss
from tests.test_gpu_xent import inputs, near, tolerances
from tests.train_testutil import Dev, close
from tests.xent_norms import errors, norm_bounds

pytestmark = pytest.mark.gpu


def run(N, D, V, dtype, softcap=0.0, kept="fp32", pad=0.0, weighted=False, seed=0):
    x, w, t = inputs(N, D, V, dtype, seed + N + V, pad=pad)
    weights = None
    if weighted:
        weights = np.random.default_rng(V).uniform(0.5, 1.5, N).astype(np.float32)
        weights[3::7] = 0.0
        x[3::7] = np.nan
    took = np.flatnonzero((t >= 0) & (t < V) & (True if weights is None else weights != 0))
    left = np.setdiff1d(np.arange(N), took)
    dx_, dw_, dt = Dev(x, dtype), Dev(w, dtype), Dev(t.astype(np.int32), "int32")
    rw = Dev(weights) if weighted else None
    gx, gw = Dev.out((N, D), kept), Dev.out((V, D), kept)
    both = [{k: Dev.out(s) for k, s in (("loss", (N,)), ("lse", (N,)), ("total", (1,)))} for _ in range(2)]
    with TokenLoss(V, D, N, dtype=dtype, dx_dtype=kept, dw_dtype=kept, softcap=softcap) as h:
        a, b = ({k: v.ptr for k, v in o.items()} for o in both)
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, dw=gw.ptr, row_weights=rw.ptr if rw else 0, **a)
        h.forward(N, dx_.ptr, dw_.ptr, dt.ptr, row_weights=rw.ptr if rw else 0, **b)
        h.synchronize()
    clean = np.zeros_like(x)
    clean[took] = x[took]
    ref = token_loss(clean, w, t, weights, softcap)
    row, bx, bw = tolerances(clean[took], w, ref, dtype, softcap, V)
    dx, dw = gx.get(), gw.get()
    assert np.all(dx[left] == 0)
    close(dx[took], ref["dx"][took], bx, kept, "dx")
    close(dw, ref["dw"], bw, kept, "dw")
    near(dx, ref["dx"], dtype, kept, bx, "dx")
    near(dw, ref["dw"], dtype, kept, bw, "dw")
    for o in both:
        loss, lse = o["loss"].get(), o["lse"].get()
        assert np.all(loss[left] == 0) and np.all(lse[left] == 0)
        close(loss[took], ref["loss"][took], row, "fp32", "loss")
        close(lse[took], ref["lse"][took], row, "fp32", "lse")
        # (the total is 64-bit sums of losses that are off by less than these)
        close(o["total"].get(), ref["total"], (ref["g"] * row).sum() + 2.0 ** -23 * ref["total"], "fp32", "total")
        if dtype == "fp32" and kept == "fp32":
            off = errors({"loss": loss[took], "lse": lse[took], "dx": dx[took], "dw": dw}, ref)
            for k, most in norm_bounds(clean[took], w, ref, softcap).items():
                assert off[k] <= most, (k, off[k] / most)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
# logits in tiles of 128 x 32, 128 x 128 and 256 x 256: of one stage of the sum, and of four
@pytest.mark.parametrize("N,D,V", [(150, 64, 900), (40, 200, 900), (2100, 40, 1000), (1500, 200, 2100),
                                   (300, 40, 16500), (700, 200, 12000)])
def test_logits(gpu_lib, N, D, V, softcap, dtype):
    run(N, D, V, dtype, softcap, pad=0.1 if D == 200 else 0.0, weighted=D == 40)


@pytest.mark.parametrize("N,D,V,dtype,kept,softcap", [
    (1500, 200, 16500, "bf16", "fp32", 0.0),    # dx in 128 x 128, split, dw in 128 x 128
    (520, 392, 8300, "fp32", "fp32", 0.0),      # dx in 128 x 128, split, dw in 128 x 128
    (520, 1001, 13000, "bf16", "bf16", 0.0),    # dx in 128 x 128, split, dw in 256 x 256
    (520, 1000, 13000, "bf16", "bf16", 30.0),   # dx in 128 x 128, split, dw in 256 x 256
    (520, 1000, 13000, "fp32", "fp32", 0.0),    # dx in 128 x 128, split, dw in 256 x 256
    (4200, 1032, 2100, "bf16", "fp32", 30.0),   # dx in 128 x 128, split, dw in 128 x 128, split
    (2100, 392, 4100, "fp32", "fp32", 0.0),     # dx in 128 x 128, split, dw in 192 x 256, split
    (13000, 1000, 520, "bf16", "bf16", 0.0),    # dx in 256 x 256, dw in 128 x 128, split
    (13000, 1001, 520, "fp32", "fp32", 30.0),   # dx in 256 x 256, dw in 128 x 128, split
    (4200, 136, 4100, "bf16", "fp32", 0.0),     # dx in 128 x 128, split, dw in 128 x 128, split
    (3000, 136, 2100, "fp32", "fp32", 0.0),     # dx in 128 x 128, split, dw in 128 x 128, split
    (200, 392, 16500, "bf16", "bf16", 0.0),     # dx in 128 x 128, split, dw in 192 x 256
    (200, 392, 16500, "fp32", "fp32", 20.0),    # dx in 128 x 128, split, dw in 192 x 256
    (9000, 1800, 300, "bf16", "fp32", 0.0),     # dx in 192 x 256, dw in 128 x 128, split
    (700, 1032, 13200, "fp32", "bf16", 0.0),    # dx in 192 x 256, split, dw in 128 x 128
])
def test_gradients(gpu_lib, N, D, V, dtype, kept, softcap):
    run(N, D, V, dtype, softcap, kept, pad=0.1 if N % 1000 else 0.0)


@pytest.mark.parametrize("N,D,V,dtype,kept,softcap", [
    (200, 200, 33000, "bf16", "fp32", 0.0),    # dw in 256 x 256, whole
    (200, 200, 33000, "fp32", "fp32", 0.0),
    (13000, 392, 4100, "bf16", "fp32", 0.0),   # dw in 256 x 256, split
    (1500, 392, 8300, "fp32", "fp32", 0.0),
    (6500, 1800, 300, "bf16", "fp32", 0.0),    # dx in 256 x 256, whole
    (6500, 1800, 300, "fp32", "fp32", 0.0),
    (4200, 392, 13000, "bf16", "fp32", 0.0),   # dx in 256 x 256, split
    (4200, 392, 4100, "fp32", "fp32", 0.0),
    (200, 136, 33000, "bf16", "fp32", 20.0),   # dw in 192 x 256, whole
    (1500, 136, 13000, "bf16", "fp32", 0.0),   # dw in 192 x 256, split
    (520, 136, 13000, "fp32", "fp32", 0.0),
    (9000, 1000, 300, "bf16", "bf16", 0.0),    # dx in 192 x 256, whole
    (9000, 1000, 300, "fp32", "fp32", 0.0),
    (13000, 136, 2100, "bf16", "fp32", 0.0),   # dx in 192 x 256, split
    (13000, 136, 520, "fp32", "fp32", 0.0),
])
def test_gradients_of_large_tiles(gpu_lib, N, D, V, dtype, kept, softcap):
    run(N, D, V, dtype, softcap, kept, seed=2)


# the small shapes' precision: losses and gradients of products in two planes each
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("N,D,V", [
    (64, 64, 64), (65, 128, 256), (130, 72, 300), (257, 96, 513), (33, 200, 1000), (300, 544, 130),
    (31, 256, 2049), (100, 1030, 70), (700, 264, 777), (200, 136, 1000), (1, 2048, 500), (16, 512, 32000),
])
def test_fp32_is_fp32(gpu_lib, N, D, V, softcap):
    run(N, D, V, "fp32", softcap, seed=1)
