"""Gradient sets on the device: norm, clipping and AdamW against the float64
restatement (oracle/train.py).

Tolerances: the norm is summed in 64 bits, so fp32's half step covers it; clip
is a coefficient in fp32 and one product (3 roundings with the result's);
AdamW's m and v are an fma, a product or two and the coefficients' roundings (4
of the absolute terms), its update three products, a root and a quotient over
them (16)."""
import numpy as np
import pytest

from mixlab_amd import _lib
from oracle import train as ot
from tests.train_testutil import U32, Dev, as_kept, close

pytestmark = pytest.mark.gpu

SETS = {
    "one": [1], "small": [3, 1, 0, 64, 7], "block": [64 * 128] * 12 + [64 * 4, 64, 64],
    "odd": [513 * 77, 5, 16384, 16385, 32767, 1], "many": [17] * 700 + [100003],
}


def _set(name, dtype, seed=0, size=1e-2):
    rng = np.random.default_rng(seed)
    return [as_kept(rng.standard_normal(n, dtype=np.float32) * np.float32(size), dtype)
            for n in SETS[name]]


def _flat(arrays, dtype="fp32", shift=0):
    """One flat buffer and each tensor's pointer into it, as a trainer keeps them."""
    whole = np.concatenate([a.reshape(-1) for a in arrays]) if arrays else np.zeros(0, np.float32)
    d = Dev(whole, dtype, shift)
    item, at, ptrs = d.np_dtype.itemsize, 0, []
    for a in arrays:
        ptrs.append(d.ptr + at * item)
        at += a.size
    return d, ptrs


@pytest.mark.parametrize("name", SETS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_norm_and_clip(gpu_lib, name, dtype, shift):
    from mixlab_amd.train import GradientSet

    grads = _set(name, dtype)
    norm = ot.global_norm(grads)
    with GradientSet(SETS[name], dtype) as s:
        g, gp = _flat(grads, dtype, shift)
        out, op = _flat([np.zeros_like(a) for a in grads], dtype, shift)
        n = Dev.out((1,))
        s.bind(gp, clipped=op)
        s.norm(n.ptr)
        s.synchronize()
        close(n.get(), [norm], 0, "fp32", "norm")
        for limit in (norm / 3, norm * 3):
            s.clip(limit, n.ptr)
            s.synchronize()
            coef = ot.clip_coef(norm, limit)
            want = coef * np.concatenate(grads).astype(np.float64)
            close(out.get(), want, 3 * U32 * np.abs(want), dtype, "clipped")
            assert np.array_equal(g.get(), np.concatenate(grads))
        s.bind(gp)  # in place
        s.clip(norm * 3)
        s.synchronize()
        assert np.array_equal(g.get(), np.concatenate(grads))
        s.clip(norm / 3)
        s.synchronize()
        want = ot.clip_coef(norm, norm / 3) * np.concatenate(grads).astype(np.float64)
        close(g.get(), want, 3 * U32 * np.abs(want), dtype, "in place")


def test_norm_of_large_and_tiny_values(gpu_lib):
    """Squares beyond fp32's range, both ways."""
    from mixlab_amd.train import GradientSet

    for size in (1e30, 1e-30, 1e-40):
        a = (np.random.default_rng(1).standard_normal(1000) * size).astype(np.float32)
        with GradientSet([600, 400]) as s:
            g, gp = _flat([a[:600], a[600:]])
            n = Dev.out((1,))
            s.bind(gp)
            s.norm(n.ptr)
            s.synchronize()
            close(n.get(), [ot.global_norm([a])], 1.4e-45, "fp32", "norm")


def _adam_state(name, seed=3):
    rng = np.random.default_rng(seed)
    ps = [0.1 * rng.standard_normal(n, dtype=np.float32) for n in SETS[name]]
    ms = [1e-3 * rng.standard_normal(n, dtype=np.float32) for n in SETS[name]]
    vs = [np.square(1e-3 * rng.standard_normal(n, dtype=np.float32)) for n in SETS[name]]
    return ps, ms, vs


@pytest.mark.parametrize("name", ["one", "small", "block", "odd", "many"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("max_norm", [0.0, 0.05])
def test_adamw(gpu_lib, name, dtype, max_norm):
    """Three steps in a row from step 0 on, with decay for every other tensor."""
    from mixlab_amd.train import GradientSet

    sizes = SETS[name]
    decay = [float(i % 2) for i in range(len(sizes))]
    ps, ms, vs = _adam_state(name)
    lr, b1, b2, eps, wd = 1e-2, 0.9, 0.999, 1e-8, 0.1
    with GradientSet(sizes, dtype, decay=decay) as s:
        (p, pp), (m, mp), (v, vp) = _flat(ps), _flat(ms), _flat(vs)
        p16, p16p = _flat([np.zeros_like(a) for a in ps], "bf16")
        step, norm, skipped = Dev(np.zeros(1, np.int64), "int64"), Dev.out((1,)), Dev.out((1,), np.int32)
        whole_decay = np.concatenate([np.full(n, w) for n, w in zip(sizes, decay)])
        for t in (1, 2, 3):
            grads = _set(name, dtype, seed=t)
            g, gp = _flat(grads, dtype)
            s.bind(gp, params=pp, m=mp, v=vp, params_bf16=p16p)
            before = [a.get().astype(np.float64) for a in (p, m, v)]
            s.adamw(lr, b1, b2, eps, wd, max_norm, step.ptr, norm.ptr, skipped.ptr)
            s.synchronize()
            n = ot.global_norm(grads)
            close(norm.get(), [n], 0, "fp32", "norm")
            gw = ot.clip_coef(n, max_norm) * np.concatenate(grads).astype(np.float64)
            want = ot.adamw(*before, gw, t, lr, b1, b2, eps, whole_decay * wd)
            close(m.get(), want[1], 4 * U32 * (np.abs(before[1]) + np.abs(gw)), "fp32", "m")
            close(v.get(), want[2], 4 * U32 * np.abs(want[2]), "fp32", "v")
            # (an error of m's relative to its terms goes into the update whole)
            big = (b1 * np.abs(before[1]) + (1 - b1) * np.abs(gw)) / (1 - b1 ** t)
            update = lr * big / (np.sqrt(want[2] / (1 - b2 ** t)) + eps)
            close(p.get(), want[0], 16 * U32 * update + 2 * U32 * np.abs(before[0]), "fp32", "p")
            close(p16.get(), p.get(), 0, "bf16", "bf16 copy")
            assert step.get()[0] == t and skipped.get()[0] == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_tensors_out_of_step(gpu_lib, dtype):
    """Gradients, outputs and state that start at different places between two
    vectors' boundaries give what aligned ones give."""
    from mixlab_amd.train import GradientSet

    sizes = [4099, 20003, 2]
    rng = np.random.default_rng(8)
    grads = [as_kept(rng.standard_normal(n, dtype=np.float32), dtype) for n in sizes]
    ps, ms, vs = ([np.abs(rng.standard_normal(n, dtype=np.float32)) for n in sizes] for _ in range(3))
    got = []
    for shifts in ((0, 0, 0, 0, 0, 0), (1, 2, 3, 1, 2, 1), (3, 1, 0, 3, 3, 3)):
        with GradientSet(sizes, dtype) as s:
            lists = [[Dev(a, t, shift=k) for a in arrays] for arrays, t, k in zip(
                (grads, grads, ps, ms, vs, ps), (dtype, dtype, "fp32", "fp32", "fp32", "bf16"), shifts)]
            step = Dev(np.zeros(1, np.int64), "int64")
            s.bind(*[[d.ptr for d in one] for one in lists])
            s.clip(0.25)
            s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, 0.25, step.ptr)
            s.synchronize()
            got.append([d.get() for one in lists for d in one])
    for other in got[1:]:
        for a, b in zip(other, got[0]):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_non_finite_gradients(gpu_lib, bad):
    """AdamW leaves everything as it was, clip copies, and the next step runs."""
    from mixlab_amd.train import GradientSet

    sizes = SETS["odd"]
    ps, ms, vs = _adam_state("odd")
    grads = _set("odd", "fp32")
    poisoned = [a.copy() for a in grads]
    poisoned[-2][123] = bad
    with GradientSet(sizes) as s:
        (p, pp), (m, mp), (v, vp) = _flat(ps), _flat(ms), _flat(vs)
        (g, gp), (good, goodp) = _flat(poisoned), _flat(grads)
        out, op = _flat([np.zeros_like(a) for a in grads])
        step, norm, skipped = Dev(np.full(1, 5, np.int64), "int64"), Dev.out((1,)), Dev.out((1,), np.int32)
        s.bind(gp, clipped=op, params=pp, m=mp, v=vp)
        s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, 1.0, step.ptr, norm.ptr, skipped.ptr)
        s.clip(0.5)
        s.synchronize()
        assert skipped.get()[0] == 1 and step.get()[0] == 5 and not np.isfinite(norm.get()[0])
        for d, a in ((p, ps), (m, ms), (v, vs)):
            assert np.array_equal(d.get(), np.concatenate(a))
        assert np.array_equal(out.get().view(np.uint32), np.concatenate(poisoned).view(np.uint32))
        s.bind(goodp, params=pp, m=mp, v=vp)
        s.adamw(1e-2, 0.9, 0.99, 1e-8, 0.1, 1.0, step.ptr, norm.ptr, skipped.ptr)
        s.synchronize()
        assert skipped.get()[0] == 0 and step.get()[0] == 6
        assert not np.array_equal(p.get(), np.concatenate(ps))


def test_step_count(gpu_lib):
    """A count past 32 bits, and one below zero, which is taken as zero."""
    from mixlab_amd.train import GradientSet

    g = _set("small", "fp32")
    ps, ms, vs = _adam_state("small")
    with GradientSet(SETS["small"]) as s:
        for start, t in ((2 ** 40, 2 ** 40 + 1), (-7, 1), (0, 1)):
            (p, pp), (m, mp), (v, vp) = _flat(ps), _flat(ms), _flat(vs)
            gd, gp = _flat(g)
            step = Dev(np.full(1, start, np.int64), "int64")
            s.bind(gp, params=pp, m=mp, v=vp)
            s.adamw(1e-2, 0.9, 0.999, 1e-8, 0.0, 0.0, step.ptr)
            s.synchronize()
            assert step.get()[0] == t
            flat = [np.concatenate(a) for a in (ps, ms, vs, g)]
            want = ot.adamw(*flat, t, 1e-2, 0.9, 0.999, 1e-8, 0.0)
            size = (0.9 * np.abs(flat[1]) + 0.1 * np.abs(flat[3])) / (1 - 0.9 ** t)
            update = 1e-2 * size / (np.sqrt(want[2] / (1 - 0.999 ** t)) + 1e-8)
            close(p.get(), want[0], 16 * U32 * update + 2 * U32 * np.abs(flat[0]), "fp32", "p")


def test_mixed_types_and_equal_bits(gpu_lib):
    from mixlab_amd.train import GradientSet

    sizes, types = [5000, 333, 70001], ["bf16", "fp32", "bf16"]
    rng = np.random.default_rng(2)
    arrays = [as_kept(rng.standard_normal(n, dtype=np.float32), t) for n, t in zip(sizes, types)]
    devs = [Dev(a, t, shift=i) for i, (a, t) in enumerate(zip(arrays, types))]
    with GradientSet(sizes, types) as s:
        s.bind([d.ptr for d in devs])
        n1, n2 = Dev.out((1,)), Dev.out((1,))
        s.norm(n1.ptr)
        s.norm(n2.ptr)
        s.synchronize()
        close(n1.get(), [ot.global_norm(arrays)], 0, "fp32", "norm")
        assert n1.get()[0] == n2.get()[0]


def test_refusals(gpu_lib):
    from mixlab_amd.train import GradientSet

    a = Dev(np.zeros(64, np.float32))
    step = Dev(np.zeros(1, np.int64), "int64")
    E = _lib.MixMoEError
    with GradientSet([8, 8]) as s:
        with pytest.raises(E, match="tensor 1: grads overlaps tensor 0's grads|tensor 0: grads overlaps"):
            s.bind([a.ptr, a.ptr])
    with GradientSet([16, 0]) as s:
        with pytest.raises(E, match="before mxm_grads_bind"):
            s.norm(a.ptr)
        with pytest.raises(E, match="tensor 0: grads is NULL"):
            s.bind([0, 0])
        with pytest.raises(E, match="tensor 0: grads is not aligned"):
            s.bind([a.ptr + 2, 0])
        with pytest.raises(E, match="tensor 0: clipped overlaps tensor 0's grads"):
            s.bind([a.ptr, 0], clipped=[a.ptr + 4, 0])
        with pytest.raises(E, match="overlaps"):
            s.bind([a.ptr, 0], params=[a.ptr + 64, 0], m=[a.ptr + 128, 0], v=[a.ptr + 128, 0])
        with pytest.raises(E, match="bound together"):
            s.bind([a.ptr, 0], params=[a.ptr, 0])
        with pytest.raises(E, match="needs params"):
            s.bind([a.ptr, 0], params_bf16=[a.ptr, 0])
        with pytest.raises(ValueError):
            s.bind([a.ptr])
        s.bind([a.ptr, 0])
        with pytest.raises(E, match="norm must be non-NULL"):
            s.norm(0)
        for limit in (0.0, -1.0, float("nan"), float("inf")):
            with pytest.raises(E, match="max_norm"):
                s.clip(limit)
        ok = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, max_norm=0.0, step=step.ptr)
        with pytest.raises(E, match="params, m and v are bound"):
            s.adamw(**ok)
        for k, v in [("lr", -1.0), ("beta1", 1.0), ("beta2", -0.1), ("eps", 0.0),
                     ("weight_decay", float("nan")), ("max_norm", -1.0), ("step", 0),
                     ("step", step.ptr + 4)]:
            with pytest.raises(E):
                s.adamw(**dict(ok, **{k: v}))
