"""What the creation of residual norms and gradient sets refuses, and calls on
handles that are none: argument errors come before any device call (CPU)."""
from __future__ import annotations

import ctypes

import pytest

from mixlab_amd import _lib

F32, BF16 = _lib.MXM_DTYPE_F32, _lib.MXM_DTYPE_BF16
BRANCH, POST, NORM, SIG = (_lib.MXM_RESNORM_BRANCH, _lib.MXM_RESNORM_POST_NORM,
                           _lib.MXM_RESNORM_NORM, _lib.MXM_RESNORM_GATE_SIGMOID)


def _create(D=64, rows=8, dtypes=(F32,) * 5, flags=BRANCH | NORM, gate=0, gate_rows=1, eps=1e-5,
            stream_of=0, n=10):
    lib = _lib.load()
    vals = [D, rows, *dtypes, flags, gate, gate_rows]
    return lib.mxm_resnorm_create((ctypes.c_int64 * 10)(*vals), n, eps, stream_of)


@pytest.mark.parametrize("kw,want", [
    (dict(n=9), "requires D,maxRows"),
    (dict(D=0), "invalid dimensions"), (dict(D=16385), "invalid dimensions"),
    (dict(rows=-1), "invalid dimensions"), (dict(rows=2 ** 30 + 1), "invalid dimensions"),
    (dict(dtypes=(F32, F32, F32, F32, 0)), "dtype 0 unsupported"),
    (dict(dtypes=(3, F32, F32, F32, F32)), "dtype 3 unsupported"),
    (dict(flags=BRANCH | 64), "unknown flags"), (dict(flags=0), "needs MXM_RESNORM_BRANCH or"),
    (dict(flags=NORM | POST), "need MXM_RESNORM_BRANCH"), (dict(flags=NORM, gate=1), "need MXM_RESNORM_BRANCH"),
    (dict(gate=3), "unsupported gate"), (dict(flags=BRANCH | SIG), "needs a gate"),
    (dict(gate=1, gate_rows=0), "gateRows"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(stream_of=987654321), "not a live handle"),
])
def test_resnorm_create_refuses(kw, want):
    assert _create(**kw) == 0
    msg = _lib.last_error()
    assert msg.startswith("RESIDUAL_NORM") and want in msg, msg


def _grads(sizes, dtypes, decay=None, n=None, stream_of=0):
    lib = _lib.load()
    k = max(1, len(sizes))
    return lib.mxm_grads_create((ctypes.c_int64 * k)(*sizes), (ctypes.c_int32 * k)(*dtypes),
                                None if decay is None else (ctypes.c_float * k)(*decay),
                                len(sizes) if n is None else n, stream_of)


@pytest.mark.parametrize("args,want", [
    (dict(sizes=[], dtypes=[]), "at least one tensor"),
    (dict(sizes=[4, -1], dtypes=[F32, F32]), "tensor 1: size -1 out of range"),
    (dict(sizes=[2 ** 40, 1], dtypes=[F32, F32]), "tensor 1: size 1 out of range"),
    (dict(sizes=[4], dtypes=[0]), "dtype 0 unsupported"),
    (dict(sizes=[4], dtypes=[BF16], decay=[float("nan")]), "decay is not finite"),
    (dict(sizes=[4], dtypes=[BF16], stream_of=987654321), "not a live handle"),
])
def test_grads_create_refuses(args, want):
    assert _grads(**args) == 0
    msg = _lib.last_error()
    assert msg.startswith("GRADIENT_SET") and want in msg, msg


def test_dead_handles():
    lib, h = _lib.load(), 987654321
    out = ctypes.c_void_p()
    assert lib.mxm_resnorm_forward(h, 1, *[None] * 8) == _lib.MXM_ERR_OP
    assert lib.mxm_resnorm_backward(h, 1, *[None] * 14) == _lib.MXM_ERR_OP
    assert lib.mxm_resnorm_destroy(h) == _lib.MXM_ERR_OP
    assert lib.mxm_grads_bind(h, *[None] * 6) == _lib.MXM_ERR_OP
    assert lib.mxm_grads_norm(h, None) == _lib.MXM_ERR_OP
    assert lib.mxm_grads_clip(h, 1.0, None) == _lib.MXM_ERR_OP
    assert lib.mxm_grads_adamw(h, *[0.1] * 6, None, None, None) == _lib.MXM_ERR_OP
    assert lib.mxm_grads_destroy(h) == _lib.MXM_ERR_OP
    assert lib.mxm_stream(h, ctypes.byref(out)) == _lib.MXM_ERR_OP
    assert lib.mxm_synchronize(h) == _lib.MXM_ERR_OP
    assert "invalid handle" in _lib.last_error()


def test_constants_match_the_header():
    from tests.test_abi import _defines

    d = _defines()
    names = [k for k in d if k.startswith(("MXM_RESNORM_", "MXM_GATE_"))]
    assert len(names) == 9
    for k in names:
        assert d[k] == getattr(_lib, k), k
