"""Residual norms and gradient sets past 2^31 elements: the far end against the
restatement on its own rows."""
import ctypes

import numpy as np
import pytest

from mixlab_amd import _lib
from mixlab_amd.workloads import bf16_bits
from oracle import train as ot
from tests.train_testutil import U32, as_kept, close, from_bits

pytestmark = pytest.mark.gpu


def _put(buf, at, bits):
    bits = np.ascontiguousarray(bits)
    _lib.check(_lib.load().mxm_memcpy_h2d(buf.value + at, bits.ctypes.data, bits.nbytes), "h2d")


def _get(buf, at, n):
    out = np.empty(n, np.uint16)
    _lib.check(_lib.load().mxm_memcpy_d2h(out.ctypes.data, buf.value + at, out.nbytes), "d2h")
    return from_bits(out)


def test_rows_past_32_bit_offsets(gpu_lib):
    """140,000 bf16 rows of 16384 (2.3e9 elements), in place; the last three rows."""
    from mixlab_amd.train import ResidualNorm

    N, D, k = 140_000, 16384, 3
    rng = np.random.default_rng(0)
    v = {n: as_kept(rng.standard_normal((k, D), dtype=np.float32), "bf16") for n in ("x", "delta", "dh", "dy")}
    far = (N - k) * D * 2
    bufs = {n: _lib.DeviceBuffer(N * D * 2) for n in v}
    tol = (D / 64 + 40) * U32
    with ResidualNorm(D, N, "bf16", "bf16", "bf16", grad_dtype="bf16", post_norm=True) as r:
        def put():
            for n, a in v.items():
                assert gpu_lib.hipMemset(ctypes.c_void_p(bufs[n].value), 0, ctypes.c_size_t(N * D * 2)) == 0
                _put(bufs[n], far, bf16_bits(a))
        put()
        r.forward(N, bufs["x"].value, bufs["delta"].value, bufs["x"].value, bufs["delta"].value)
        r.synchronize()
        h, y = (_get(bufs[n], far, k * D).reshape(k, D) for n in ("x", "delta"))
        f = {n: a.astype(np.float64) for n, a in v.items()}
        want, share = ot.resnorm_sum(f["x"], f["delta"], post_norm=True)
        close(h, want, tol * np.abs(share), "bf16", "h")
        want = ot.rms_norm(h.astype(np.float64))
        close(y, want, tol * np.abs(want), "bf16", "y")
        assert not np.any(_get(bufs["x"], 0, 4 * D))  # zero rows stay zero
        put()
        r.backward(N, bufs["x"].value, bufs["delta"].value, bufs["dh"].value, bufs["dy"].value,
                   bufs["dh"].value, bufs["dy"].value)
        r.synchronize()
        args = (f["x"], f["delta"], f["dh"], f["dy"])
        want = ot.resnorm_backward(*args, post_norm=True)
        size = ot.resnorm_backward(*args, post_norm=True, absolute=True)
        for n, key in (("dh", "dx"), ("dy", "d_delta")):
            close(_get(bufs[n], far, k * D).reshape(k, D), want[key], tol * size[key], "bf16", key)


def test_a_gradient_of_over_2_31_elements(gpu_lib):
    from mixlab_amd.train import GradientSet

    n, k = 2 ** 31 + 5, 1000
    tail = as_kept(np.random.default_rng(1).standard_normal(k, dtype=np.float32), "bf16")
    buf, norm = _lib.DeviceBuffer(n * 2), _lib.DeviceBuffer(4)
    assert gpu_lib.hipMemset(ctypes.c_void_p(buf.value), 0, ctypes.c_size_t(n * 2)) == 0
    _put(buf, (n - k) * 2, bf16_bits(tail))
    want = ot.global_norm([tail])
    with GradientSet([n], "bf16") as s:
        s.bind([buf.value])
        s.clip(want / 4, norm.value)
        s.synchronize()
        close(norm.download(np.float32, (1,)), [want], 0, "fp32", "norm")
        scaled = ot.clip_coef(want, want / 4) * tail.astype(np.float64)
        close(_get(buf, (n - k) * 2, k), scaled, 3 * U32 * np.abs(scaled), "bf16", "clipped")
