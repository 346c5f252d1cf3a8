"""Helpers of the tests of residual norms and gradient sets: arrays on the
device, and the tolerances of fp32 evaluations."""
from __future__ import annotations

import numpy as np

from mixlab_amd import _lib
from mixlab_amd.workloads import bf16_bits

U32 = 2.0 ** -24   # half a step of fp32, relative
UBF = 2.0 ** -8    # of bf16


def from_bits(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def as_kept(a, dtype):
    """fp32 values as a tensor of `dtype` holds them."""
    a = np.ascontiguousarray(a, np.float32)
    return from_bits(bf16_bits(a)).reshape(a.shape) if dtype == "bf16" else a


class Dev:
    """An array on the device, `shift` elements past an allocation's start and
    with `guard` sentinel elements behind it."""

    SENTINEL = 0x5A

    def __init__(self, a, dtype="fp32", shift=0, guard=64):
        a = np.ascontiguousarray(a)
        if dtype == "bf16":
            bits = bf16_bits(np.ascontiguousarray(a, np.float32))
        elif dtype == "fp32":
            bits = np.ascontiguousarray(a, np.float32)
        else:
            bits = a
        self.dtype, self.shape, self.np_dtype = dtype, a.shape, bits.dtype
        self.size, self.shift, self.guard = bits.size, shift, guard
        whole = np.full((shift + bits.size + guard) * bits.itemsize, self.SENTINEL, np.uint8)
        whole[shift * bits.itemsize:(shift + bits.size) * bits.itemsize] = bits.reshape(-1).view(np.uint8)
        self.buf = _lib.DeviceBuffer.from_array(whole)
        self.ptr = self.buf.value + shift * bits.itemsize

    @classmethod
    def out(cls, shape, dtype="fp32", shift=0):
        """An output, full of sentinels (NaN-free patterns that no test computes)."""
        kind = {"bf16": np.uint16, "fp32": np.float32}.get(dtype, dtype)
        n = int(np.prod(shape))
        d = cls(np.zeros(0, np.float32), "fp32")
        d.dtype, d.shape, d.np_dtype = dtype, tuple(shape), np.dtype(kind)
        d.size, d.shift, d.guard = n, shift, 64
        item = d.np_dtype.itemsize
        d.buf = _lib.DeviceBuffer.from_array(np.full((shift + n + 64) * item, cls.SENTINEL, np.uint8))
        d.ptr = d.buf.value + shift * item
        return d

    def put(self, a):
        """Other values of the same type (fp32 or whole numbers) in place."""
        a = np.ascontiguousarray(a, self.np_dtype)
        assert a.size == self.size and self.dtype != "bf16"
        if a.size:
            _lib.check(_lib.load().mxm_memcpy_h2d(self.ptr, a.ctypes.data, a.nbytes), "mxm_memcpy_h2d")

    def get(self):
        """The values (bf16 widened to fp32); whatever lies around them is untouched."""
        item = self.np_dtype.itemsize
        raw = self.buf.download(np.uint8, ((self.shift + self.size + self.guard) * item,))
        assert np.all(raw[:self.shift * item] == self.SENTINEL), "written before the tensor"
        assert np.all(raw[(self.shift + self.size) * item:] == self.SENTINEL), "written behind it"
        v = raw[self.shift * item:(self.shift + self.size) * item].view(self.np_dtype).reshape(self.shape)
        return from_bits(v) if self.dtype == "bf16" else v.copy()


def close(got, want, bound, dtype="fp32", what=""):
    """|got - want| <= bound, and half a step of the type it is kept in."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.asarray(bound, np.float64) + (UBF if dtype == "bf16" else U32) * np.abs(want) * 1.01 + 1e-37
    off = np.abs(got - want)
    bad = ~(off <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, off / tol, 0)), off.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, at {i} got {got[i]!r} want "
                             f"{want[i]!r} tolerance {tol[i] if tol.shape else tol!r}")
