"""The residual norm on the device, both directions, against its float64
restatement (oracle/train.py).

Tolerances: an fp32 evaluation of these formulas is off by at most c * 2^-24
times the same sums over absolute values (the restatement's absolute=True),
with c the length of the longest chain of roundings: the sums over a row go
over at most D / 64 terms a lane and a tree (D / 64 + 16), each is used in a
handful of products (24), and column sums add at most a chunk's rows and the
chunks' slices (N / 1024 + 8 rows, then 64 additions).  Outputs kept in 16 bits
are off by half a step more."""
import numpy as np
import pytest

from mixlab_amd import _lib
from oracle import train as ot
from tests.train_testutil import U32, Dev, as_kept, close

pytestmark = pytest.mark.gpu


def _row_c(D):
    return (D / 64 + 40) * U32


def _col_c(N, D):
    return _row_c(D) + (2 * (N / 1024 + 8) + 64) * U32


def _case(seed, N, D, stream="fp32", delta="fp32", out="fp32", scale="fp32", grad="fp32", post=True,
          norm=True, gate=None, gate_rows=1, sigmoid=False, scales=True):
    rng = np.random.default_rng(seed)

    def randn(*shape):
        return rng.standard_normal(shape, dtype=np.float32)

    v = dict(x=as_kept(randn(N, D), stream), delta=as_kept(0.3 * randn(N, D), delta),
             dh=as_kept(randn(N, D), grad), dy=as_kept(randn(N, D), grad),
             h=as_kept(randn(N, D), stream))
    if scales:
        v["branch_scale"] = as_kept(0.5 + 0.1 * randn(D), scale)
        if post:
            v["post_scale"] = as_kept(1 + 0.1 * randn(D), scale)
        if norm:
            v["norm_scale"] = as_kept(1 + 0.1 * randn(D), scale)
    if gate:
        v["gate"] = as_kept(randn(-(-N // gate_rows), D if gate == "channel" else 1), scale)
    return v


def _handle(N, D, stream="fp32", delta="fp32", out="fp32", scale="fp32", grad="fp32", post=True,
            norm=True, gate=None, gate_rows=1, sigmoid=False, scales=True, **kw):
    from mixlab_amd.train import ResidualNorm

    return ResidualNorm(D, N, stream_dtype=stream, delta_dtype=delta, out_dtype=out,
                        scale_dtype=scale, grad_dtype=grad, post_norm=post, norm=norm, gate=gate,
                        gate_rows=gate_rows, gate_sigmoid=sigmoid, **kw)


def _scales(v, types, shift=0):
    d = {k: Dev(v[k], types, shift) for k in ("post_scale", "branch_scale", "norm_scale", "gate") if k in v}
    return d, {k: t.ptr for k, t in d.items()}


def run_forward(v, N, D, shift=0, rows=None, handle=None, **c):
    stream, out = c.get("stream", "fp32"), c.get("out", "fp32")
    x, delta = Dev(v["x"], stream, shift), Dev(v["delta"], c.get("delta", "fp32"), shift)
    h, y = Dev.out((N, D), stream, shift), Dev.out((N, D), out, shift)
    hold, ptrs = _scales(v, c.get("scale", "fp32"), shift)
    r = handle or _handle(N, D, **c)
    r.forward(N if rows is None else rows, x.ptr, delta.ptr, h.ptr, y.ptr if c.get("norm", True) else 0,
              **ptrs)
    r.synchronize()
    return h, y


def check_forward(v, h, y, N, D, c):
    gate = v.get("gate")
    args = (v.get("post_scale"), v.get("branch_scale"), gate, c.get("gate_rows", 1),
            c.get("sigmoid", False), c.get("post", True))
    want, share = ot.resnorm_sum(v["x"].astype(np.float64), v["delta"].astype(np.float64), *args)
    close(h, want, _row_c(D) * np.abs(share) + U32 * np.abs(want), c.get("stream", "fp32"), "h")
    if c.get("norm", True):
        want = ot.rms_norm(h.astype(np.float64), v.get("norm_scale"))
        close(y, want, _row_c(D) * np.abs(want), c.get("out", "fp32"), "y")


def run_backward(v, N, D, shift=0, rows=None, handle=None, use_dh=True, **c):
    grad, norm = c.get("grad", "fp32"), c.get("norm", True)
    delta = Dev(v["delta"], c.get("delta", "fp32"), shift)
    h = Dev(v["h"], c.get("stream", "fp32"), shift)
    dh, dy = Dev(v["dh"], grad, shift), Dev(v["dy"], grad, shift)
    out = dict(dx=Dev.out((N, D), grad, shift), d_delta=Dev.out((N, D), grad, shift))
    hold, ptrs = _scales(v, c.get("scale", "fp32"), shift)
    G = 0
    out["d_scale"] = Dev.out((D,), shift=shift)
    kw = dict(d_branch_scale=out["d_scale"].ptr)
    if c.get("post", True):
        out["d_post"] = Dev.out((D,), shift=shift)
        kw["d_post_scale"] = out["d_post"].ptr
    if norm:
        out["d_w"] = Dev.out((D,), shift=shift)
        kw["d_norm_scale"] = out["d_w"].ptr
    if "gate" in v:
        out["d_gate"] = Dev.out(v["gate"].shape, shift=shift)
        kw["d_gate"] = out["d_gate"].ptr
    r = handle or _handle(N, D, **c)
    r.backward(N if rows is None else rows, h.ptr if norm else 0, delta.ptr, dh.ptr if use_dh else 0,
               dy.ptr if norm else 0, out["dx"].ptr, out["d_delta"].ptr, **ptrs, **kw)
    r.synchronize()
    return {k: t.get() for k, t in out.items()}


def check_backward(v, got, N, D, c, use_dh=True):
    norm, grad = c.get("norm", True), c.get("grad", "fp32")
    f = lambda k: v[k].astype(np.float64)  # noqa: E731
    args = (f("h") if norm else None, f("delta"), f("dh") if use_dh else None, f("dy") if norm else None,
            v.get("post_scale"), v.get("branch_scale"), v.get("gate"), c.get("gate_rows", 1),
            c.get("sigmoid", False), c.get("post", True), v.get("norm_scale"))
    want, size = ot.resnorm_backward(*args), ot.resnorm_backward(*args, absolute=True)
    assert set(got) == set(want) - (set() if c.get("post", True) else {"d_post"})
    # (a gate's rows add up to gate_rows more terms in chunks' and slices' order)
    for k in got:
        if k in ("dx", "d_delta"):
            close(got[k], want[k], _row_c(D) * size[k], grad, k)
        else:
            close(got[k], want[k], _col_c(N, D) * size[k], "fp32", k)


SHAPES = [(1, 1), (2, 3), (5, 63), (1, 64), (37, 66), (3, 127), (9, 257), (130, 512), (33, 544),
          (4, 1000), (300, 1024), (17, 2048), (2, 2052), (5, 4100), (3, 8191), (2, 16384)]


@pytest.mark.parametrize("N,D", SHAPES)
@pytest.mark.parametrize("types", ["fp32", "bf16", "mixed"])
def test_widths(gpu_lib, N, D, types):
    c = {"fp32": {}, "bf16": dict(stream="bf16", delta="bf16", out="bf16", scale="bf16", grad="bf16"),
         "mixed": dict(out="bf16", gate="row", sigmoid=True)}[types]
    v = _case(N * 100 + D, N, D, **c)
    h, y = run_forward(v, N, D, **c)
    check_forward(v, h.get(), y.get(), N, D, c)
    check_backward(v, run_backward(v, N, D, **c), N, D, c)


@pytest.mark.parametrize("gate", ["row", "channel"])
@pytest.mark.parametrize("N,gate_rows", [(1, 1), (7, 1), (64, 3), (64, 7), (65, 64), (200, 1000),
                                         (1000, 333), (2500, 2), (2500, 1200)])
@pytest.mark.parametrize("D", [8, 260])
def test_gates(gpu_lib, gate, N, gate_rows, D):
    c = dict(gate=gate, gate_rows=gate_rows, sigmoid=(N + D) % 2 == 0)
    v = _case(N + gate_rows + D, N, D, **c)
    h, y = run_forward(v, N, D, **c)
    check_forward(v, h.get(), y.get(), N, D, c)
    check_backward(v, run_backward(v, N, D, **c), N, D, c)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("scales", [False, True])
@pytest.mark.parametrize("D", [96, 1030])
def test_parts(gpu_lib, post, norm, scales, D):
    """Each of the norms and scales left out."""
    c = dict(post=post, norm=norm, scales=scales)
    v = _case(7, 21, D, **c)
    h, y = run_forward(v, 21, D, **c)
    check_forward(v, h.get(), y.get(), 21, D, c)
    check_backward(v, run_backward(v, 21, D, **c), 21, D, c)
    if norm:
        check_backward(v, run_backward(v, 21, D, use_dh=False, **c), 21, D, c, use_dh=False)


@pytest.mark.parametrize("N,D", [(6, 100), (6, 1024), (2, 4098)])
@pytest.mark.parametrize("stream", ["fp32", "bf16"])
def test_norm_alone(gpu_lib, N, D, stream):
    """Without a branch: the norm at a block's entry, and its backward, which adds
    the stream's own gradient."""
    from mixlab_amd.train import ResidualNorm

    v = _case(11, N, D, stream=stream)
    with ResidualNorm(D, N, stream_dtype=stream, out_dtype="bf16", branch=False) as r:
        x, y = Dev(v["x"], stream), Dev.out((N, D), "bf16")
        w, dh, dy = Dev(v["norm_scale"]), Dev(v["dh"]), Dev(v["dy"])
        dx, dw = Dev.out((N, D)), Dev.out((D,))
        r.forward(N, x.ptr, y=y.ptr, norm_scale=w.ptr)
        r.backward(N, x.ptr, dh=dh.ptr, dy=dy.ptr, dx=dx.ptr, norm_scale=w.ptr, d_norm_scale=dw.ptr)
        r.synchronize()
        want = ot.rms_norm(v["x"].astype(np.float64), v["norm_scale"])
        close(y.get(), want, _row_c(D) * np.abs(want), "bf16", "y")
        args = (v["x"].astype(np.float64), None, v["dh"].astype(np.float64),
                v["dy"].astype(np.float64))
        g = ot.resnorm_backward(*args, norm_scale=v["norm_scale"])
        b = ot.resnorm_backward(*args, norm_scale=v["norm_scale"], absolute=True)
        close(dx.get(), g["dx"], _row_c(D) * b["dx"], "fp32", "dx")
        close(dw.get(), g["d_w"], _col_c(N, D) * b["d_w"], "fp32", "d_w")


@pytest.mark.parametrize("D", [64, 544, 2048])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_unaligned(gpu_lib, D, shift):
    """Tensors that start between two vectors' boundaries."""
    c = dict(out="bf16", gate="channel", gate_rows=4)
    v = _case(shift, 10, D, **c)
    h, y = run_forward(v, 10, D, shift=shift, **c)
    check_forward(v, h.get(), y.get(), 10, D, c)
    check_backward(v, run_backward(v, 10, D, shift=shift, **c), 10, D, c)


@pytest.mark.parametrize("D", [64, 515, 2048])
def test_rows_behind_are_left(gpu_lib, D):
    """Fewer rows than the handle was made for: the rest keeps what it held, and no
    rows at all give zero gradients of the scales."""
    N, rows = 40, 23
    v = _case(3, N, D)
    with _handle(N, D) as r:
        h, y = run_forward(v, N, D, rows=rows, handle=r)
        part = {k: (a[:rows] if a.ndim == 2 else a) for k, a in v.items()}
        untouched = np.full(4, Dev.SENTINEL, np.uint8).view(np.float32)[0]
        assert np.all(h.get()[rows:] == untouched) and np.all(y.get()[rows:] == untouched)
        check_forward(part, h.get()[:rows], y.get()[:rows], rows, D, {})
        got = run_backward(v, N, D, rows=rows, handle=r)
        assert np.all(got["dx"][rows:] == untouched) and np.all(got["d_delta"][rows:] == untouched)
        got["dx"], got["d_delta"] = got["dx"][:rows], got["d_delta"][:rows]
        check_backward(part, got, rows, D, {})
        none = run_backward(v, N, D, rows=0, handle=r)
        for k in ("d_scale", "d_post", "d_w"):
            assert np.all(none[k] == 0)
        assert np.all(none["dx"] == untouched)


@pytest.mark.parametrize("D", [96, 1024])
def test_zero_and_non_finite_rows(gpu_lib, D):
    """A zero row has finite results; NaN and infinity stay in their own rows."""
    N = 8
    v = _case(9, N, D)
    for k in ("x", "delta", "h", "dh", "dy"):
        v[k][2] = 0
    h, y = run_forward(v, N, D)
    check_forward(v, h.get(), y.get(), N, D, {})
    check_backward(v, run_backward(v, N, D), N, D, {})
    good = run_backward(v, N, D)
    bad = {k: a.copy() for k, a in v.items()}
    bad["delta"][4, 5], bad["x"][6, 1], bad["h"][6, 1] = np.nan, np.inf, np.inf
    h2, y2 = run_forward(bad, N, D)
    keep = [n for n in range(N) if n not in (4, 6)]
    assert np.array_equal(h2.get()[keep], h.get()[keep]) and np.array_equal(y2.get()[keep], y.get()[keep])
    assert np.isnan(h2.get()[4]).all() and np.isnan(y2.get()[4]).all()
    got = run_backward(bad, N, D)
    for k in ("dx", "d_delta"):
        assert np.array_equal(got[k][keep], good[k][keep])
    assert np.isnan(got["d_scale"]).any()


@pytest.mark.parametrize("N,D", [(1025, 520), (1300, 767), (1100, 1000), (1030, 1021), (3, 5000),
                                 (2, 9001)])
@pytest.mark.parametrize("types", ["fp32", "bf16"])
def test_more_rows_and_wide_rows(gpu_lib, N, D, types):
    """Rows in a wave past the few, and rows over 512 threads."""
    c = dict(gate="channel", gate_rows=7, sigmoid=True)
    if types == "bf16":
        c.update(stream="bf16", delta="bf16", out="bf16", grad="bf16")
    v = _case(N + D, N, D, **c)
    h, y = run_forward(v, N, D, **c)
    check_forward(v, h.get(), y.get(), N, D, c)
    check_backward(v, run_backward(v, N, D, **c), N, D, c)


@pytest.mark.parametrize("rows", [1, 700, 1024, 1025, 3000])
def test_one_handle_for_many_sizes(gpu_lib, rows):
    """The workspace made for the most rows holds any fewer, whatever shape they take."""
    c = dict(gate="channel", gate_rows=100)
    v = _case(rows, rows, 600, **c)
    with _handle(3000, 600, **c) as r:
        check_backward(v, run_backward(v, rows, 600, handle=r, **c), rows, 600, c)


@pytest.mark.parametrize("N,D", [(5000, 64), (3000, 1030), (2100, 2048)])
def test_many_rows_and_equal_bits(gpu_lib, N, D):
    """More chunks than workgroups fit at once; two runs agree bit for bit."""
    c = dict(gate="channel", gate_rows=600)
    v = _case(N, N, D, **c)
    with _handle(N, D, **c) as r:
        a = run_backward(v, N, D, handle=r, **c)
        b = run_backward(v, N, D, handle=r, **c)
        h, y = run_forward(v, N, D, handle=r, **c)
    check_backward(v, a, N, D, c)
    check_forward(v, h.get(), y.get(), N, D, c)
    for k in a:
        assert np.array_equal(a[k].view(np.uint32), b[k].view(np.uint32)), k


@pytest.mark.parametrize("D", [64, 1030])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_in_place(gpu_lib, D, dtype):
    """h over x, dx over dh, d_delta over dy give what separate buffers give."""
    N, c = 19, dict(stream=dtype, delta=dtype, out=dtype, grad=dtype, gate="channel", gate_rows=5)
    v = _case(1, N, D, **c)
    h, y = run_forward(v, N, D, **c)
    g = run_backward(v, N, D, **c)
    with _handle(N, D, **c) as r:
        hold, ptrs = _scales(v, "fp32")
        x, delta = Dev(v["x"], dtype), Dev(v["delta"], dtype)
        r.forward(N, x.ptr, delta.ptr, x.ptr, delta.ptr, **ptrs)
        r.synchronize()
        assert np.array_equal(x.get(), h.get()) and np.array_equal(delta.get(), y.get())
        hh, delta = Dev(v["h"], dtype), Dev(v["delta"], dtype)
        dh, dy = Dev(v["dh"], dtype), Dev(v["dy"], dtype)
        r.backward(N, hh.ptr, delta.ptr, dh.ptr, dy.ptr, dh.ptr, dy.ptr, **ptrs)
        r.synchronize()
        assert np.array_equal(dh.get(), g["dx"]) and np.array_equal(dy.get(), g["d_delta"])


@pytest.mark.parametrize("N,D", [(7, 20), (33, 100), (9, 300), (21, 1000)])
@pytest.mark.parametrize("gate", [None, "channel"])
def test_no_epsilon_and_an_infinite_gate(gpu_lib, N, D, gate):
    """eps 0, numbers of rows that leave threads without one, and an infinite gate in
    the last group: only what reads it is not finite."""
    c = dict(gate=gate, gate_rows=4)
    v = _case(N, N, D, **c)
    from mixlab_amd.train import ResidualNorm
    with ResidualNorm(D, N, out_dtype="fp32", post_norm=True, eps=0.0, gate=gate, gate_rows=4) as r:
        good = run_backward(v, N, D, handle=r, **c)
        assert all(np.isfinite(a).all() for a in good.values())
        if gate:
            v["gate"][-1, 3] = np.inf
            bad = run_backward(v, N, D, handle=r, **c)
            rows = (N - 1) // 4 * 4
            assert np.array_equal(bad["dx"], good["dx"])
            assert np.array_equal(bad["d_delta"][:rows], good["d_delta"][:rows])
            other = np.arange(D) != 3
            for k in ("d_scale", "d_post"):
                assert np.array_equal(bad[k][other], good[k][other]) and not np.isfinite(bad[k][3])
            assert np.array_equal(bad["d_gate"], good["d_gate"])


def test_refusals(gpu_lib):
    N, D = 4, 32
    v = _case(0, N, D)
    with _handle(N, D) as r:
        x, d, h, y = Dev(v["x"]), Dev(v["delta"]), Dev.out((N, D)), Dev.out((N, D))
        for kw, text in [(dict(rows=5), "rows 5 out of range"), (dict(rows=-1), "rows -1 out of range"),
                         (dict(x=0), "x must be non-NULL"), (dict(delta=0), "delta must be non-NULL"),
                         (dict(h=0), "h must be non-NULL"), (dict(y=0), "y must be non-NULL"),
                         (dict(x=x.ptr + 2), "x is not aligned")]:
            a = dict(rows=N, x=x.ptr, delta=d.ptr, h=h.ptr, y=y.ptr)
            a.update(kw)
            with pytest.raises(_lib.MixMoEError, match=text):
                r.forward(**a)
        with pytest.raises(_lib.MixMoEError, match="dy must be non-NULL"):
            r.backward(N, x.ptr, d.ptr, x.ptr, 0, h.ptr, y.ptr)
        with pytest.raises(_lib.MixMoEError, match="dx must be non-NULL"):
            r.backward(N, x.ptr, d.ptr, x.ptr, x.ptr, 0, y.ptr)
        with pytest.raises(_lib.MixMoEError, match="d_gate given without a gate"):
            r.backward(N, x.ptr, d.ptr, x.ptr, x.ptr, h.ptr, y.ptr, d_gate=h.ptr)
    with _handle(N, D, backward=False, post=False) as r:
        with pytest.raises(_lib.MixMoEError, match="MXM_RESNORM_BACKWARD"):
            r.backward(N, x.ptr, d.ptr, x.ptr, x.ptr, h.ptr, y.ptr)
        with pytest.raises(_lib.MixMoEError, match="without MXM_RESNORM_POST_NORM"):
            r.forward(N, x.ptr, d.ptr, h.ptr, y.ptr, post_scale=x.ptr)
    assert gpu_lib.mxm_resnorm_forward(r.handle or 987654, 1, *[None] * 8) == _lib.MXM_ERR_OP
