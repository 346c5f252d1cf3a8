"""Calls on residual norms and gradient sets in orders, at values and over
buffers that a program can come to."""
import numpy as np
import pytest

from mixlab_amd import _lib, moe
from mixlab_amd.train import GradientSet, MoEBlockTrainer, ResidualNorm
from oracle import train as ot
from tests.test_gpu_resnorm import _case, _col_c, _handle, _row_c, run_backward, run_forward
from tests.test_gpu_train_streams import Graph
from tests.train_testutil import U32, Dev, as_kept, close

pytestmark = pytest.mark.gpu


def test_replayed_update_after_a_bind_without_params(gpu_lib):
    """A captured AdamW step reads the pointers bound last: with none for params it
    updates nothing, and goes on once they are bound again."""
    sizes = [1000, 0, 3]
    rng = np.random.default_rng(0)
    with GradientSet(sizes) as s:
        g, p, m, v = ([Dev(rng.random(n, dtype=np.float32)) for n in sizes] for _ in range(4))
        ptrs = [[d.ptr for d in one] for one in (g, p, m, v)]
        step, skipped, norm = Dev(np.zeros(1, np.int64), "int64"), Dev.out((1,), np.int32), Dev.out((1,))

        def state():
            s.synchronize()
            return [d.get() for one in (p, m, v) for d in one]

        s.bind(ptrs[0], params=ptrs[1], m=ptrs[2], v=ptrs[3])
        graph = Graph(gpu_lib, s.stream(), lambda: s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, 0.0, step.ptr,
                                                           norm.ptr, skipped.ptr))
        graph.replay()
        once = state()
        assert step.get()[0] == 1 and skipped.get()[0] == 0
        s.bind(ptrs[0])
        graph.replay()
        for a, b in zip(state(), once):
            assert np.array_equal(a, b)
        assert step.get()[0] == 1 and skipped.get()[0] == 1
        close(norm.get(), [ot.global_norm([d.get() for d in g])], 0, "fp32", "norm")
        s.bind(ptrs[0], params=ptrs[1], m=ptrs[2], v=ptrs[3])
        graph.replay()
        assert not np.array_equal(state()[0], once[0])
        assert step.get()[0] == 2 and skipped.get()[0] == 0
        graph.close()


def _check_backward(v, got, D, size_bound, **kw):
    """Row and column gradients within size_bound of the sums over absolute values."""
    f = lambda k: v[k].astype(np.float64)  # noqa: E731
    args = (f("h"), f("delta"), None, f("dy"), v["post_scale"], v["branch_scale"], v.get("gate"))
    want = ot.resnorm_backward(*args, post_norm=True, norm_scale=v["norm_scale"], **kw)
    size = ot.resnorm_backward(*args, post_norm=True, norm_scale=v["norm_scale"], absolute=True, **kw)
    for k in want:
        close(got[k], want[k], size_bound * size[k], v["dtype"] if k in ("dx", "d_delta") else "fp32", k)


@pytest.mark.parametrize("N,D", [(5, 64), (9, 300), (4, 1024), (3, 2049), (2, 9000)])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-5), (1e17, 1e-5), (1e-16, 0.0)])
@pytest.mark.parametrize("gate", [None, "row", "channel"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_backward_of_large_and_tiny_rows(gpu_lib, N, D, size, eps, gate, dtype):
    """Rows whose 1 / rms has a cube outside fp32's range (the sums' squares are
    inside it) keep both terms of their gradients.  dh is left out and dy as large
    as the rows, so that every gradient is far from the range's ends."""
    c = dict(stream=dtype, delta=dtype, grad=dtype, gate=gate)
    v = _case(N + D, N, D, **c)
    for k in ("h", "delta", "dy"):
        v[k] = as_kept(v[k] * np.float32(size), dtype)
    with ResidualNorm(D, N, stream_dtype=dtype, delta_dtype=dtype, out_dtype="fp32", grad_dtype=dtype,
                      post_norm=True, eps=eps, gate=gate) as r:
        got = run_backward(v, N, D, handle=r, use_dh=False, **c)
    _check_backward(dict(v, dtype=dtype), got, D, _col_c(N, D), eps=eps)


@pytest.mark.parametrize("N,D", [(6, 64), (6, 300), (5, 1024), (3, 2051)])
@pytest.mark.parametrize("gate", [None, "row", "channel"])
def test_non_finite_branch_without_a_post_norm(gpu_lib, N, D, gate):
    """d_delta does not depend on delta then: an infinite or NaN element of it only
    shows in the sums that read it."""
    c = dict(post=False, norm=False, gate=gate, gate_rows=2)
    v = _case(N, N, D, **c)
    good = run_backward(v, N, D, **c)
    bad = dict(v, delta=v["delta"].copy())
    bad["delta"][1, 5], bad["delta"][2, 9] = np.inf, np.nan
    got = run_backward(bad, N, D, **c)
    for k in ("dx", "d_delta"):
        assert np.array_equal(got[k], good[k]), k
    other = ~np.isin(np.arange(D), (5, 9))
    assert np.array_equal(got["d_scale"][other], good["d_scale"][other])
    assert not np.isfinite(got["d_scale"][[5, 9]]).any()


@pytest.mark.parametrize("gate,gate_rows", [("row", 1), ("row", 7), ("row", 40), ("channel", 1), ("channel", 7),
                                            ("channel", 40)])
@pytest.mark.parametrize("N,D", [(40, 64), (40, 544), (9, 2051)])
@pytest.mark.parametrize("post", [False, True])
def test_gradient_of_a_saturated_gate(gpu_lib, N, D, gate, gate_rows, post):
    """A sigmoid's slope a (1 - a) keeps its digits where a is next to 1: gates from
    -60 to 60 (slopes from 9e-27 on).  The exponential and the slope add about ten
    roundings, within the handful that the bound counts."""
    c = dict(post=post, norm=False, gate=gate, gate_rows=gate_rows, sigmoid=True)
    v = _case(N + D, N, D, **c)
    v["gate"] = np.random.default_rng(D).uniform(-60, 60, v["gate"].shape).astype(np.float32)
    got = run_backward(v, N, D, **c)
    f = lambda k: v[k].astype(np.float64)  # noqa: E731
    args = (None, f("delta"), f("dh"), None, v.get("post_scale"), v["branch_scale"], v["gate"], gate_rows,
            True, post)
    want, size = ot.resnorm_backward(*args), ot.resnorm_backward(*args, absolute=True)
    for k in got:
        close(got[k], want[k], (_row_c(D) if k == "d_delta" else _col_c(N, D)) * size[k], "fp32", k)


def test_gates_of_any_value(gpu_lib):
    """Infinite and NaN gates through the sigmoid, both zeros, and the largest."""
    N, D = 8, 96
    c = dict(post=True, norm=False, gate="row", gate_rows=1, sigmoid=True)
    v = _case(1, N, D, **c)
    v["gate"][:, 0] = (np.inf, -np.inf, 0.0, -0.0, 3e38, -3e38, np.nan, 1.0)
    got = run_backward(v, N, D, **c)
    with np.errstate(over="ignore"):
        a = 1.0 / (1.0 + np.exp(-v["gate"].astype(np.float64)))
    assert np.isnan(got["d_delta"][6]).all() and np.isnan(got["d_gate"][6])
    assert np.all(got["d_delta"][[1, 5]] == 0) and np.all(got["d_gate"][[0, 1, 4, 5]] == 0)
    keep = [n for n in range(N) if n != 6]
    args = [x[keep].astype(np.float64) for x in (v["delta"], v["dh"], v["gate"])]
    want = ot.resnorm_backward(None, args[0], args[1], None, v["post_scale"], v["branch_scale"], a[keep],
                               1, False, True)
    size = ot.resnorm_backward(None, args[0], args[1], None, v["post_scale"], v["branch_scale"], a[keep],
                               1, False, True, absolute=True)
    close(got["d_delta"][keep], want["d_delta"], _row_c(D) * size["d_delta"], "fp32", "d_delta")


@pytest.mark.parametrize("max_norm", [0.0, 1.0, 1e30])
def test_norm_beyond_fp32(gpu_lib, max_norm):
    """Finite gradients whose norm is infinite as fp32: *norm says so, and so do the
    step that changes nothing and the clip that copies."""
    g = np.array([3e38, 0.0, -3e38, 1.0, 2.0], np.float32)
    old = [np.full(5, x, np.float32) for x in (0.5, 0.25, 0.125)]
    with GradientSet([5]) as s:
        d, out, (p, m, v) = Dev(g), Dev.out((5,)), (Dev(a) for a in old)
        step, norm, skipped = Dev(np.full(1, 7, np.int64), "int64"), Dev.out((1,)), Dev.out((1,), np.int32)
        s.bind([d.ptr], [out.ptr], [p.ptr], [m.ptr], [v.ptr])
        s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, max_norm, step.ptr, norm.ptr, skipped.ptr)
        s.synchronize()
        assert norm.get()[0] == np.inf and skipped.get()[0] == 1 and step.get()[0] == 7
        for a, b in zip((p, m, v), old):
            assert np.array_equal(a.get(), b)
        if max_norm:
            s.clip(max_norm, norm.ptr)
            s.synchronize()
            assert norm.get()[0] == np.inf and np.array_equal(out.get(), g)


def test_largest_norm_of_fp32(gpu_lib):
    """A norm next to fp32's largest value is finite: the step runs and clips.  The
    coefficient is a subnormal, off by 2^-150, half of fp32's smallest step."""
    g = np.array([2e38, -2e38, 1e38, 1.5e38, 0.5], np.float32)
    n = ot.global_norm([g])
    coef = ot.clip_coef(n, 1.0)
    bound = (2.0 ** -150 + 3 * U32 * coef) * np.abs(g.astype(np.float64))
    with GradientSet([5]) as s:
        d, out, (p, m, v) = Dev(g), Dev.out((5,)), (Dev(np.zeros(5, np.float32)) for _ in range(3))
        step, norm, skipped = Dev(np.zeros(1, np.int64), "int64"), Dev.out((1,)), Dev.out((1,), np.int32)
        s.bind([d.ptr], [out.ptr], [p.ptr], [m.ptr], [v.ptr])
        s.clip(1.0, norm.ptr)
        s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.0, 1.0, step.ptr, norm.ptr, skipped.ptr)
        s.synchronize()
        close(norm.get(), [n], 0, "fp32", "norm")
        assert skipped.get()[0] == 0 and step.get()[0] == 1
        close(out.get(), coef * g.astype(np.float64), bound, "fp32", "clipped")
        close(m.get(), 0.1 * coef * g.astype(np.float64), bound, "fp32", "m")


@pytest.mark.parametrize("size", [1e-40, 1e-38, 1e-44])
@pytest.mark.parametrize("n", [3, 1000, 200000])
def test_norm_of_subnormal_gradients(gpu_lib, size, n):
    """Subnormal gradients are not flushed, and neither is a subnormal norm: half of
    fp32's smallest step, or of the value's."""
    a = (np.random.default_rng(n).standard_normal(n) * size).astype(np.float32)
    assert np.any(a)
    with GradientSet([n]) as s:
        d, norm = Dev(a), Dev.out((1,))
        s.bind([d.ptr])
        s.norm(norm.ptr)
        s.synchronize()
        want = ot.global_norm([a])
        assert abs(float(norm.get()[0]) - want) <= max(2.0 ** -150, U32 * want) * (1 + 1e-9)


N, D = 6, 24
ITEM = {"fp32": 4, "bf16": 2}


def _spare(dtype="fp32", rows=N):
    return Dev.out((rows, D), dtype)


@pytest.mark.parametrize("types", ["fp32", "mixed"])
def test_overlaps_of_a_forward(gpu_lib, types):
    """An output in the place of an input of its type is fine; the rest is refused
    before anything runs."""
    b = "bf16" if types == "mixed" else "fp32"
    with ResidualNorm(D, N, delta_dtype=b, out_dtype="fp32", post_norm=True, gate="channel", gate_rows=4) as r:
        x, delta, h, y = _spare(rows=3 * N), _spare(b, 3 * N), _spare(), _spare(rows=3 * N)
        s, g = _spare(rows=4), _spare(rows=4)
        ok = dict(rows=N, x=x.ptr, delta=delta.ptr, h=h.ptr, y=y.ptr, branch_scale=s.ptr, gate=g.ptr)
        bad = [("h overlaps x", dict(h=x.ptr + 4)), ("h overlaps x", dict(x=x.ptr + 4 * D, h=x.ptr)),
               ("y overlaps x", dict(y=x.ptr + 4 * (N * D - 1))),
               ("h overlaps y", dict(h=y.ptr + 4 * D)), ("h overlaps branch_scale", dict(branch_scale=h.ptr + 8)),
               ("y overlaps gate", dict(gate=y.ptr + 4 * D)),
               ("y overlaps post_scale", dict(post_scale=y.ptr + 4 * (N - 1) * D)),
               ("y overlaps norm_scale", dict(norm_scale=y.ptr))]
        if types == "mixed":
            bad += [("y overlaps delta", dict(y=delta.ptr)), ("h overlaps delta", dict(h=delta.ptr))]
        for text, kw in bad:
            with pytest.raises(_lib.MixMoEError, match=text):
                r.forward(**dict(ok, **kw))
        good = [dict(h=x.ptr), dict(y=x.ptr), dict(h=x.ptr, y=y.ptr), dict(x=x.ptr, h=x.ptr + 4 * N * D),
                dict(delta=x.ptr) if types == "fp32" else {}, dict(post_scale=s.ptr, norm_scale=s.ptr, gate=s.ptr)]
        if types == "fp32":
            good += [dict(h=delta.ptr), dict(y=delta.ptr), dict(h=delta.ptr, y=x.ptr)]
        for kw in good:
            r.forward(**dict(ok, **kw))
        r.synchronize()


def test_overlaps_of_a_backward(gpu_lib):
    with ResidualNorm(D, N, out_dtype="fp32", post_norm=True, gate="channel", gate_rows=4) as r, \
            ResidualNorm(D, N, scale_dtype="bf16", gate="row", gate_rows=2) as rb:
        h, delta, dh, dy, dx, dd = (_spare(rows=2 * N) for _ in range(6))
        v = {k: _spare(rows=2) for k in ("post", "scale", "w", "gate", "dp", "ds", "dw", "dg")}
        ok = dict(rows=N, h=h.ptr, delta=delta.ptr, dh=dh.ptr, dy=dy.ptr, dx=dx.ptr, d_delta=dd.ptr,
                  post_scale=v["post"].ptr, branch_scale=v["scale"].ptr, norm_scale=v["w"].ptr,
                  gate=v["gate"].ptr, d_post_scale=v["dp"].ptr, d_branch_scale=v["ds"].ptr,
                  d_norm_scale=v["dw"].ptr, d_gate=v["dg"].ptr)
        for text, kw in [
                ("dx overlaps d_delta", dict(dx=dd.ptr + 4 * D)), ("dx overlaps dh", dict(dx=dh.ptr + 4)),
                ("d_delta overlaps dy", dict(d_delta=dy.ptr + 4 * D)), ("dx overlaps h", dict(h=dx.ptr + 4 * D)),
                ("d_delta overlaps gate", dict(d_delta=v["gate"].ptr)),
                ("d_post_scale overlaps d_branch_scale", dict(d_post_scale=v["ds"].ptr)),
                ("d_branch_scale overlaps post_scale", dict(d_branch_scale=v["post"].ptr)),
                ("d_norm_scale overlaps branch_scale", dict(d_norm_scale=v["scale"].ptr)),
                ("d_gate overlaps post_scale", dict(d_gate=v["post"].ptr)),
                ("d_gate overlaps gate", dict(d_gate=v["gate"].ptr + 4 * D)),
                ("d_norm_scale overlaps dy|d_norm_scale overlaps d", dict(d_norm_scale=dy.ptr))]:
            with pytest.raises(_lib.MixMoEError, match=text):
                r.backward(**dict(ok, **kw))
        both = dict(rows=N, h=h.ptr, delta=delta.ptr, dh=dh.ptr, dy=dy.ptr, dx=dx.ptr, d_delta=dd.ptr,
                    branch_scale=v["scale"].ptr, gate=v["gate"].ptr)
        for text, kw in [("d_branch_scale overlaps branch_scale", dict(d_branch_scale=v["scale"].ptr)),
                         ("d_gate overlaps gate", dict(d_gate=v["gate"].ptr))]:
            with pytest.raises(_lib.MixMoEError, match=text):  # bf16 under fp32
                rb.backward(**dict(both, **kw))
        for kw in (dict(dx=dh.ptr), dict(d_delta=dy.ptr), dict(d_delta=delta.ptr, dx=h.ptr), dict(dh=dy.ptr),
                   dict(d_delta=dh.ptr, dx=dy.ptr)):
            r.backward(**dict(ok, **kw))
        r.synchronize()


@pytest.mark.parametrize("N,D,gate_rows", [(40, 64, 1), (40, 300, 7), (700, 64, 700), (9, 1030, 2)])
def test_gradients_in_their_scales_places(gpu_lib, N, D, gate_rows):
    """The scales' and the gate's gradients over the scales and the gate themselves."""
    c = dict(gate="channel", gate_rows=gate_rows, sigmoid=True)
    v = _case(N, N, D, **c)
    want = run_backward(v, N, D, **c)
    t = {k: Dev(v[k]) for k in ("h", "delta", "dh", "dy", "post_scale", "branch_scale", "norm_scale", "gate")}
    with ResidualNorm(D, N, out_dtype="fp32", post_norm=True, gate="channel", gate_rows=gate_rows,
                      gate_sigmoid=True) as r:
        r.backward(N, dx=t["dh"].ptr, d_delta=t["dy"].ptr, d_post_scale=t["post_scale"].ptr,
                   d_branch_scale=t["branch_scale"].ptr, d_gate=t["gate"].ptr,
                   d_norm_scale=t["norm_scale"].ptr, **{k: d.ptr for k, d in t.items()})
        r.synchronize()
    for k, place in (("dx", "dh"), ("d_delta", "dy"), ("d_post", "post_scale"), ("d_scale", "branch_scale"),
                     ("d_w", "norm_scale"), ("d_gate", "gate")):
        assert np.array_equal(t[place].get(), want[k]), k


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("gate", ["row", "channel"])
def test_trainer_gates_on_the_device(gpu_lib, dtype, gate):
    """A gate on the device in the compute's type gives what step_host gives for its
    values in fp32; its gradient is fp32 in both."""
    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": 4, "top_k": 2})
    B, T, width = 2, 15, 96
    rng = np.random.default_rng(3)
    x, d_out = (rng.standard_normal((B * T, width), dtype=np.float32) for _ in range(2))
    g = rng.standard_normal((B, width) if gate == "channel" else (B, 1), dtype=np.float32)
    with MoEBlockTrainer(spec, B, T, width, 1.0, post_norm=True, gate=gate, gate_rows=T,
                         compute_dtype=dtype) as tr:
        tr.set_weights([np.ones(m.shape) if len(m.shape) == 1 else 0.05 * rng.standard_normal(m.shape)
                        for m in tr.metas])
        want = tr.step_host(x, d_out, 0.0, g)
        bx, bd, bo, bg, dg = Dev(x), Dev(d_out), Dev.out(x.shape), Dev(g, dtype), Dev.out(g.shape)
        tr.forward(bx.ptr, bo.ptr, bg.ptr)
        tr.backward(bd.ptr, bd.ptr, dg.ptr)
        assert tr.update(0.0)
        assert np.array_equal(bo.get(), want["out"]) and np.array_equal(bd.get(), want["dx"])
        assert np.array_equal(dg.get(), want["d_gate"])


@pytest.mark.parametrize("kw", [dict(lr=1e39), dict(lr=1e30, weight_decay=1e30), dict(lr=1.0, weight_decay=1e39)])
def test_rates_past_fp32(gpu_lib, kw):
    """Finite rates that are infinite in the update's fp32 are refused: they would make
    weights of zero gradient NaN."""
    with GradientSet([4]) as s:
        g, p, m, v = (Dev(np.zeros(4, np.float32)) for _ in range(4))
        step = Dev(np.zeros(1, np.int64), "int64")
        s.bind([g.ptr], params=[p.ptr], m=[m.ptr], v=[v.ptr])
        args = dict(dict(dict(lr=1e-3, weight_decay=0.0), **kw), beta1=0.9, beta2=0.99, eps=1e-8, max_norm=1.0,
                    step=step.ptr)
        with pytest.raises(_lib.MixMoEError, match="fp32"):
            s.adamw(**args)
        s.adamw(**dict(args, lr=1e30, weight_decay=1.0))
        s.synchronize()
        assert step.get()[0] == 1 and not p.get().any()


@pytest.mark.parametrize("N,D", [(9, 64), (9, 301), (5, 1030), (3, 4100)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_results_that_are_not_wanted(gpu_lib, N, D, dtype):
    """h in y's buffer, or dx in d_delta's: the later result is what is left."""
    c = dict(stream=dtype, delta=dtype, out=dtype, grad=dtype)
    v = _case(N, N, D, **c)
    y = run_forward(v, N, D, **c)[1].get()
    dd = run_backward(v, N, D, **c)["d_delta"]
    t = {k: Dev(v[k], dtype) for k in ("x", "delta", "h", "dh", "dy")}
    s = {k: Dev(v[k]) for k in ("post_scale", "branch_scale", "norm_scale")}
    scales = {k: d.ptr for k, d in s.items()}
    with _handle(N, D, **c) as r:
        for x, place in ((t["x"], Dev.out((N, D), dtype)), (t["x"], t["x"])):
            r.forward(N, x.ptr, t["delta"].ptr, place.ptr, place.ptr, **scales)
            r.synchronize()
            assert np.array_equal(place.get(), y)
        place = Dev.out((N, D), dtype)
        r.backward(N, t["h"].ptr, t["delta"].ptr, t["dh"].ptr, t["dy"].ptr, place.ptr, place.ptr, **scales)
        r.synchronize()
        assert np.array_equal(place.get(), dd)
    if dtype == "fp32":
        with _handle(N, D, out="bf16") as r:
            with pytest.raises(_lib.MixMoEError, match="h overlaps y"):
                r.forward(N, t["x"].ptr, t["delta"].ptr, place.ptr, place.ptr, **scales)
