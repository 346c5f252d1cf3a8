"""A training step around the MoE op, on libmixmoe.

``ResidualNorm`` is what stands between a block's branch and the next block
(post norm, scale, gate, residual add, next norm) in both directions;
``GradientSet`` the global gradient norm, clipping and AdamW over a block's
tensors.  Both take device pointers (ints) and run asynchronously on a stream
that they can share with an op.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

from . import _lib
from .op import _DTYPES

_GATES = {None: _lib.MXM_GATE_NONE, "row": _lib.MXM_GATE_ROW, "channel": _lib.MXM_GATE_CHANNEL}


class _Handle:
    """A handle of the library: its stream, waiting for it, its release."""

    _destroy = ""

    def _open(self, handle: int) -> None:
        if not handle:
            raise _lib.MixMoEError(_lib.last_error())
        self.handle = handle

    def stream(self) -> int:
        """The hipStream_t (as an int) that the calls run on."""
        out = ctypes.c_void_p()
        _lib.check(self._lib.mxm_stream(self.handle, ctypes.byref(out)), "mxm_stream")
        return out.value or 0

    def synchronize(self) -> None:
        _lib.check(self._lib.mxm_synchronize(self.handle), "mxm_synchronize")

    def close(self) -> None:
        if getattr(self, "handle", 0):
            getattr(self._lib, self._destroy)(self.handle)
            self.handle = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


class ResidualNorm(_Handle):
    """h = x + gate * branch_scale * post_scale * z, y = norm_scale * rms(h), with
    z = rms(delta) under post_norm, else delta (include/mixmoe.h has the
    formulas).  ``share`` is the object (an op, another of these) whose stream
    the calls run on.  branch=False leaves the norm alone: y of x."""

    _destroy = "mxm_resnorm_destroy"

    def __init__(self, D: int, max_rows: int, stream_dtype: str = "fp32", delta_dtype: str = "fp32",
                 out_dtype: str = "bf16", scale_dtype: str = "fp32", grad_dtype: str = "fp32",
                 eps: float = 1e-5, branch: bool = True, post_norm: bool = False, norm: bool = True,
                 gate: Optional[str] = None, gate_rows: int = 1, gate_sigmoid: bool = False,
                 backward: bool = True, share=None):
        self._lib = _lib.init()
        flags = ((_lib.MXM_RESNORM_BRANCH if branch else 0)
                 | (_lib.MXM_RESNORM_POST_NORM if post_norm else 0)
                 | (_lib.MXM_RESNORM_NORM if norm else 0)
                 | (_lib.MXM_RESNORM_GATE_SIGMOID if gate_sigmoid else 0)
                 | (_lib.MXM_RESNORM_BACKWARD if backward else 0))
        vals = [D, max_rows, *(_DTYPES[t] for t in (stream_dtype, delta_dtype, out_dtype,
                                                    scale_dtype, grad_dtype)),
                flags, _GATES[gate], gate_rows]
        arr = (ctypes.c_int64 * len(vals))(*vals)
        self._open(self._lib.mxm_resnorm_create(arr, len(vals), float(eps),
                                                share.handle if share is not None else 0))

    def forward(self, rows: int, x: int, delta: int = 0, h: int = 0, y: int = 0,
                post_scale: int = 0, branch_scale: int = 0, gate: int = 0,
                norm_scale: int = 0) -> None:
        _lib.check(self._lib.mxm_resnorm_forward(
            self.handle, rows, x or None, delta or None, post_scale or None, branch_scale or None, gate or None,
            norm_scale or None, h or None, y or None), "mxm_resnorm_forward")

    def backward(self, rows: int, h: int = 0, delta: int = 0, dh: int = 0, dy: int = 0, dx: int = 0,
                 d_delta: int = 0, post_scale: int = 0, branch_scale: int = 0, gate: int = 0,
                 norm_scale: int = 0, d_post_scale: int = 0, d_branch_scale: int = 0,
                 d_gate: int = 0, d_norm_scale: int = 0) -> None:
        _lib.check(self._lib.mxm_resnorm_backward(
            self.handle, rows, h or None, delta or None, post_scale or None, branch_scale or None, gate or None,
            norm_scale or None, dh or None, dy or None, dx or None, d_delta or None, d_post_scale or None,
            d_branch_scale or None, d_gate or None, d_norm_scale or None), "mxm_resnorm_backward")


class GradientSet(_Handle):
    """The gradients of several tensors: their norm, clipping, AdamW.
    ``dtypes`` is one type for all or one per tensor; ``decay`` multiplies the
    weight decay of each tensor (default 1)."""

    _destroy = "mxm_grads_destroy"

    def __init__(self, sizes: Sequence[int], dtypes: Union[str, Sequence[str]] = "fp32",
                 decay: Optional[Sequence[float]] = None, share=None):
        self._lib = _lib.init()
        n = len(sizes)
        if isinstance(dtypes, str):
            dtypes = [dtypes] * n
        if len(dtypes) != n or (decay is not None and len(decay) != n):
            raise ValueError(f"{n} sizes, {len(dtypes)} dtypes"
                             + ("" if decay is None else f", {len(decay)} decays"))
        self.n = n
        cs = (ctypes.c_int64 * max(1, n))(*[int(s) for s in sizes])
        cd = (ctypes.c_int32 * max(1, n))(*[_DTYPES[t] for t in dtypes])
        cw = None if decay is None else (ctypes.c_float * max(1, n))(*decay)
        self._open(self._lib.mxm_grads_create(cs, cd, cw, n,
                                              share.handle if share is not None else 0))

    def bind(self, grads: Sequence[int], clipped: Optional[Sequence[int]] = None,
             params: Optional[Sequence[int]] = None, m: Optional[Sequence[int]] = None,
             v: Optional[Sequence[int]] = None, params_bf16: Optional[Sequence[int]] = None) -> None:
        """Device pointers, one per tensor (see mxm_grads_bind)."""
        def arr(ptrs):
            if ptrs is None:
                return None
            if len(ptrs) != self.n:
                raise ValueError(f"{len(ptrs)} pointers for {self.n} tensors")
            return (ctypes.c_void_p * self.n)(*[p or None for p in ptrs])

        _lib.check(self._lib.mxm_grads_bind(self.handle, *(arr(p) for p in (
            grads, clipped, params, m, v, params_bf16))), "mxm_grads_bind")

    def norm(self, norm: int) -> None:
        _lib.check(self._lib.mxm_grads_norm(self.handle, norm or None), "mxm_grads_norm")

    def clip(self, max_norm: float, norm: int = 0) -> None:
        _lib.check(self._lib.mxm_grads_clip(self.handle, max_norm, norm or None), "mxm_grads_clip")

    def adamw(self, lr: float, beta1: float, beta2: float, eps: float, weight_decay: float,
              max_norm: float, step: int, norm: int = 0, skipped: int = 0) -> None:
        _lib.check(self._lib.mxm_grads_adamw(self.handle, lr, beta1, beta2, eps, weight_decay,
                                             max_norm, step or None, norm or None, skipped or None),
                   "mxm_grads_adamw")
