"""What the creation of token embeddings and token losses refuses, and calls on
handles that are none: argument errors come before any device call (CPU)."""
from __future__ import annotations

import ctypes

import pytest

from mixlab_amd import _lib

F32, BF16 = _lib.MXM_DTYPE_F32, _lib.MXM_DTYPE_BF16


def _embed(V=64, D=8, rows=4, dtypes=(F32,) * 4, flags=1, scale=1.0, stream_of=0, n=8):
    vals = [V, D, rows, *dtypes, flags]
    return _lib.load().mxm_embed_create((ctypes.c_int64 * 8)(*vals), n, scale, stream_of)


def _xent(V=64, D=8, rows=4, dtypes=(F32,) * 3, flags=3, softcap=0.0, stream_of=0, n=7):
    vals = [V, D, rows, *dtypes, flags]
    return _lib.load().mxm_xent_create((ctypes.c_int64 * 7)(*vals), n, softcap, stream_of)


SIZES = [
    (dict(V=0), "invalid dimensions"), (dict(V=2 ** 24 + 1), "invalid dimensions"),
    (dict(D=0), "invalid dimensions"), (dict(D=16385), "invalid dimensions"),
    (dict(rows=-1), "invalid dimensions"), (dict(rows=2 ** 30 + 1), "invalid dimensions"),
    (dict(stream_of=987654321), "not a live handle"), (dict(flags=8), "unknown flags"),
]


@pytest.mark.parametrize("kw,want", SIZES + [
    (dict(n=7), "requires V,D,maxRows"), (dict(dtypes=(F32, 0, F32, F32)), "dtype 0 unsupported"),
    (dict(dtypes=(F32, F32, F32, 3)), "dtype 3 unsupported"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
])
def test_embed_create_refuses(kw, want):
    assert _embed(**kw) == 0
    msg = _lib.last_error()
    assert msg.startswith("TOKEN_EMBEDDING") and want in msg, msg


@pytest.mark.parametrize("kw,want", SIZES + [
    (dict(n=6), "requires V,D,maxRows"), (dict(dtypes=(0, F32, F32)), "dtype 0 unsupported"),
    (dict(dtypes=(BF16, F32, 3)), "dtype 3 unsupported"),
    (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(softcap=float("inf")), "softcap"), (dict(softcap=0.01), "softcap"), (dict(softcap=1025.0), "softcap"),
])
def test_xent_create_refuses(kw, want):
    assert _xent(**kw) == 0
    msg = _lib.last_error()
    assert msg.startswith("TOKEN_LOSS") and want in msg, msg


def test_calls_on_no_handle():
    lib = _lib.load()
    bad = 987654321
    assert lib.mxm_embed_forward(bad, 0, None, None, None) == _lib.MXM_ERR_OP
    assert lib.mxm_embed_backward(bad, 0, None, None, None, 0) == _lib.MXM_ERR_OP
    assert lib.mxm_embed_destroy(bad) == _lib.MXM_ERR_OP
    assert "TOKEN_EMBEDDING invalid handle" in _lib.last_error()
    assert lib.mxm_xent_forward(bad, 0, *[None] * 7) == _lib.MXM_ERR_OP
    assert lib.mxm_xent_backward(bad, 0, *[None] * 4, 1.0, *[None] * 5) == _lib.MXM_ERR_OP
    assert lib.mxm_xent_destroy(bad) == _lib.MXM_ERR_OP
    assert "TOKEN_LOSS invalid handle" in _lib.last_error()


def test_a_closed_object_shares_no_stream():
    from mixlab_amd.vocab import TokenEmbedding, TokenLoss

    class Closed:
        handle = 0

    with pytest.raises(ValueError, match="closed"):
        TokenEmbedding(8, 8, 1, share=Closed())
    with pytest.raises(ValueError, match="closed"):
        TokenLoss(8, 8, 1, share=Closed())


@pytest.mark.parametrize("create", [_embed, _xent])
@pytest.mark.parametrize("kw", [dict(V=_lib.MXM_VOCAB_MAX + 1), dict(D=_lib.MXM_RESNORM_MAX_D + 1),
                                dict(V=-1), dict(D=-1), dict(rows=-2 ** 62), dict(V=2 ** 62), dict(D=2 ** 62)])
def test_sizes_right_behind_the_limits(create, kw):
    assert create(**kw) == 0
    assert "invalid dimensions (V in [1,4194304], D in [1,16384], maxRows in [0,2^30])" in _lib.last_error()
