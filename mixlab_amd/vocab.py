"""The vocabulary's two ends of a training step, on libmixmoe.

``TokenEmbedding`` looks tokens up in a table and sums their gradients into one;
``TokenLoss`` is the softmax cross entropy of the last hidden rows against a
table (the same one, where they are tied), with its gradients.  Both take device
pointers (ints) and run asynchronously on a stream that they can share with an op
and with the handles of ``mixlab_amd.train``.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .op import _DTYPES
from .train import _Handle, _stream_of


class TokenEmbedding(_Handle):
    """out[n] = scale * table[tokens[n]] for a table [vocab, D] (include/mixmoe.h has
    what holds for tokens outside it).  ``share`` is the object (an op, another of
    these) whose stream the calls run on."""

    _destroy = "mxm_embed_destroy"

    def __init__(self, vocab: int, D: int, max_rows: int, table_dtype: str = "fp32",
                 out_dtype: str = "fp32", grad_dtype: str = "fp32", table_grad_dtype: str = "fp32",
                 scale: float = 1.0, backward: bool = True, share=None):
        stream_of = _stream_of(share)
        self._lib = _lib.init()
        vals = [vocab, D, max_rows,
                *(_DTYPES[t] for t in (table_dtype, out_dtype, grad_dtype, table_grad_dtype)),
                _lib.MXM_EMBED_BACKWARD if backward else 0]
        arr = (ctypes.c_int64 * len(vals))(*vals)
        self._open(self._lib.mxm_embed_create(arr, len(vals), float(scale), stream_of))

    def forward(self, rows: int, tokens: int, table: int, out: int) -> None:
        _lib.check(self._lib.mxm_embed_forward(self.handle, rows, tokens or None, table or None,
                                               out or None), "mxm_embed_forward")

    def backward(self, rows: int, tokens: int, d_out: int, d_table: int,
                 accumulate: bool = False) -> None:
        _lib.check(self._lib.mxm_embed_backward(self.handle, rows, tokens or None, d_out or None,
                                                d_table or None, 1 if accumulate else 0),
                   "mxm_embed_backward")


class TokenLoss(_Handle):
    """The weighted softmax cross entropy of x [rows, D] against weight [vocab, D], and
    its gradients (include/mixmoe.h has the formulas).  ``dtype`` is that of x and
    weight; mean divides the total by the weights' sum."""

    _destroy = "mxm_xent_destroy"

    def __init__(self, vocab: int, D: int, max_rows: int, dtype: str = "bf16", dx_dtype: str = "fp32",
                 dw_dtype: str = "fp32", softcap: float = 0.0, mean: bool = True,
                 backward: bool = True, share=None):
        stream_of = _stream_of(share)
        self._lib = _lib.init()
        vals = [vocab, D, max_rows, *(_DTYPES[t] for t in (dtype, dx_dtype, dw_dtype)),
                (_lib.MXM_XENT_MEAN if mean else 0) | (_lib.MXM_XENT_BACKWARD if backward else 0)]
        arr = (ctypes.c_int64 * len(vals))(*vals)
        self._open(self._lib.mxm_xent_create(arr, len(vals), float(softcap), stream_of))

    def forward(self, rows: int, x: int, weight: int, targets: int, row_weights: int = 0,
                loss: int = 0, lse: int = 0, total: int = 0) -> None:
        _lib.check(self._lib.mxm_xent_forward(
            self.handle, rows, x or None, weight or None, targets or None, row_weights or None,
            loss or None, lse or None, total or None), "mxm_xent_forward")

    def backward(self, rows: int, x: int, weight: int, targets: int, dx: int = 0, dw: int = 0,
                 row_weights: int = 0, d_total: float = 1.0, loss: int = 0, lse: int = 0,
                 total: int = 0) -> None:
        _lib.check(self._lib.mxm_xent_backward(
            self.handle, rows, x or None, weight or None, targets or None, row_weights or None,
            float(d_total), loss or None, lse or None, total or None, dx or None, dw or None),
            "mxm_xent_backward")
