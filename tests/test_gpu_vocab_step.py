"""The vocabulary's two ends with what stands between them, as a training program runs
them on one stream: embedding, one block, the last norm, the token loss against the
embedding's own table, and back; AdamW on all of it.  Also what programs do around
that: threads, graphs, handles that share a stream, a step's calls in any sizes."""
import threading

import numpy as np
import pytest

from mixlab_amd import _lib, moe
from mixlab_amd.train import GradientSet, MoEBlockTrainer, ResidualNorm
from mixlab_amd.vocab import TokenEmbedding, TokenLoss
from mixlab_amd.workloads import bf16_bits, round_bf16
from oracle import train as ot
from oracle.backward import forward64
from oracle.vocab import embed_backward, embed_forward, token_loss
from tests.moe_testutil import rel_l2
from tests.test_gpu_train_block import TOL, _reference, _weights
from tests.test_gpu_train_streams import Graph
from tests.train_testutil import U32, Dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,B,T,D,V,softcap", [
    ("fp32", 2, 33, 64, 90, 0.0),
    ("fp32", 1, 50, 72, 200, 6.0),
    ("bf16", 2, 40, 256, 300, 0.0),
    ("bf16", 1, 64, 136, 151, 8.0),
])
def test_training_step_on_a_tied_table(gpu_lib, dtype, B, T, D, V, softcap):
    bf16, N, scale = dtype == "bf16", B * T, 1.5
    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": 4, "top_k": 2})
    etype, act, _ = moe.moe_expert_type_and_activation(spec)
    kept = "bf16" if bf16 else "fp32"
    r = round_bf16 if bf16 else (lambda a: np.asarray(a, np.float32))
    rng = np.random.default_rng(N + V)
    tokens = rng.integers(0, V, N).astype(np.int32)
    targets = np.roll(tokens, -1).copy()
    tokens[::11] = -1
    targets[-1] = targets[::7] = -100
    table = (rng.standard_normal((V, D)) * (2.0 / np.sqrt(D))).astype(np.float32)
    wn = (1.0 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    lr, hyper = 1e-2, (0.9, 0.95, 1e-8, 0.1, 0.5)
    with MoEBlockTrainer(spec, B, T, D, 2.0, compute_dtype=dtype) as tr:
        ws = _weights(rng, tr.metas)
        tr.set_weights(ws)
        emb = TokenEmbedding(V, D, N, table_dtype=kept, scale=scale, share=tr.op)
        last = ResidualNorm(D, N, out_dtype=kept, scale_dtype="fp32", branch=False, share=tr.op)
        end = TokenLoss(V, D, N, dtype=kept, softcap=softcap, share=emb)
        opt = GradientSet([V * D, D], decay=[1.0, 0.0], share=end)
        assert emb.stream() == last.stream() == end.stream() == opt.stream() == tr.entry.stream()
        dtok, dtgt = Dev(tokens, "int32"), Dev(targets, "int32")
        master, norm_w = Dev(table), Dev(wn)
        copy = Dev(table, "bf16") if bf16 else master
        spare = Dev(wn, "bf16")
        m, v = ([Dev(np.zeros(n, np.float32)) for n in (V * D, D)] for _ in range(2))
        h0, h1, dh1, dh0, dy = (Dev.out((N, D)) for _ in range(5))
        y = Dev.out((N, D), kept)
        g_table, g_norm = Dev.out((V, D)), Dev.out((D,))
        total, norm, step = Dev.out((1,)), Dev.out((1,)), Dev(np.zeros(1, np.int64), "int64")
        opt.bind([g_table.ptr, g_norm.ptr], params=[master.ptr, norm_w.ptr], m=[b.ptr for b in m],
                 v=[b.ptr for b in v], params_bf16=[copy.ptr, spare.ptr] if bf16 else None)

        emb.forward(N, dtok.ptr, copy.ptr, h0.ptr)
        tr.forward(h0.ptr, h1.ptr)
        last.forward(N, h1.ptr, y=y.ptr, norm_scale=norm_w.ptr)
        end.backward(N, y.ptr, copy.ptr, dtgt.ptr, dx=dy.ptr, dw=g_table.ptr, total=total.ptr)
        last.backward(N, h1.ptr, dy=dy.ptr, dx=dh1.ptr, norm_scale=norm_w.ptr, d_norm_scale=g_norm.ptr)
        tr.backward(dh1.ptr, dh0.ptr)
        emb.backward(N, dtok.ptr, dh0.ptr, g_table.ptr, accumulate=True)
        opt.adamw(lr, *hyper, step.ptr, norm.ptr)
        opt.synchronize()
        top_idx = tr.op.routing()["top_idx"].astype(np.int64)
        block_grads = tr.gradients()

        # the same in 64 bits, on this routing
        w64 = r(table).astype(np.float64)
        want = {"h0": embed_forward(tokens, w64, scale)}
        f = _reference(ws, tr.metas, want["h0"].astype(np.float32), np.zeros((N, D), np.float32), 2,
                       tr.aux_weight, etype, act, False, None, 1, top_idx, bf16)
        y64 = ot.rms_norm(f["out"], wn.astype(np.float64))
        loss = token_loss(r(y64.astype(np.float32)), w64, targets, softcap=softcap)
        b = ot.resnorm_backward(f["out"], None, None, loss["dx"], norm_scale=wn.astype(np.float64))
        f = _reference(ws, tr.metas, want["h0"].astype(np.float32), b["dx"].astype(np.float32), 2,
                       tr.aux_weight, etype, act, False, None, 1, top_idx, bf16)
        want_table = embed_backward(tokens, f["dx"], V, scale, loss["dw"])

        # three stages forward and three back, each within its own tolerance
        tol = 6 * TOL[dtype]
        assert abs(total.get()[0] - loss["total"][0]) <= tol * abs(loss["total"][0])
        assert rel_l2(dy.get(), loss["dx"]) <= tol
        assert rel_l2(dh0.get(), f["dx"]) <= tol
        assert rel_l2(g_norm.get(), b["d_w"]) <= tol
        got_table = g_table.get()
        assert rel_l2(got_table, want_table) <= tol
        for meta, a, c in zip(tr.metas, block_grads, f["grads"]):
            assert rel_l2(a, c) <= (4 if meta.name == "router_w" else 1) * tol, meta.name

        if not bf16:
            # against differences of the whole loss, along directions of all its weights
            named = {mm.name: w.astype(np.float64) for mm, w in zip(tr.metas, ws)}
            mats = [w.astype(np.float64) for mm, w in zip(tr.metas, ws) if mm.name.startswith("expert_")]

            def value(tab, wnorm):
                x = embed_forward(tokens, tab, scale)
                ff = forward64(ot.rms_norm(x, named["moe_norm_scale"]), named["router_w"],
                               [mats[i:i + 3] for i in range(0, len(mats), 3)], top_idx, etype, act, 0.0)
                out = token_loss(ot.rms_norm(x + ff["delta"], wnorm), tab, targets, softcap=softcap)
                return out["total"][0] + tr.aux_weight * ff["aux"]

            for k in range(3):
                du = np.random.default_rng(k).standard_normal((V, D))
                dn = np.random.default_rng(k).standard_normal(D) if k else np.zeros(D)
                e = 1e-5
                diff = (value(w64 + e * du, wn + e * dn) - value(w64 - e * du, wn - e * dn)) / (2 * e)
                along = (got_table * du).sum() + (g_norm.get() * dn).sum()
                size = np.linalg.norm(got_table) * np.linalg.norm(du) + np.linalg.norm(g_norm.get()) * np.linalg.norm(dn)
                # (of two vectors' product, their lengths'; the differences' own error is
                # e^2 of a third derivative and 2^-53 of the loss over e)
                assert abs(diff - along) <= tol * size + 1e-8

        # the optimizer's step on it
        gn = ot.global_norm([got_table, g_norm.get()])
        assert abs(norm.get()[0] - gn) <= 2 ** -23 * gn
        p, _, _ = ot.adamw(table, 0.0, 0.0, ot.clip_coef(gn, 0.5) * got_table.astype(np.float64), 1, lr,
                           0.9, 0.95, 1e-8, 0.1)
        assert np.max(np.abs(master.get() - p)) <= 2 ** -18 * lr + 2 ** -23 * np.max(np.abs(p))
        if bf16:
            assert np.array_equal(copy.get(), round_bf16(master.get()))
        assert tr.update(lr)
        for h in (opt, end, last, emb):
            h.close()


class Ends:
    """An embedding and a loss on one table, with their buffers."""

    def __init__(self, N, D, V, dtype, softcap=0.0, share=None, weighted=False):
        self.N, self.D, self.V, self.dtype = N, D, V, dtype
        self.emb = TokenEmbedding(V, D, N, table_dtype=dtype, out_dtype=dtype, scale=0.5, share=share)
        self.loss = TokenLoss(V, D, N, dtype=dtype, softcap=softcap, share=self.emb)
        self.tok, self.tgt = (Dev(np.zeros(N, np.int32), "int32") for _ in range(2))
        self.table = Dev(np.zeros((V, D), np.float32), dtype)
        self.h, self.dh, self.dw = Dev.out((N, D), dtype), Dev.out((N, D)), Dev.out((V, D))
        self.per, self.lse, self.total = Dev.out((N,)), Dev.out((N,)), Dev.out((1,))
        self.rw = Dev(np.ones(N, np.float32)) if weighted else None

    def fill(self, seed, rows=None):
        rng = np.random.default_rng(seed)
        tok, tgt = (rng.integers(-self.V // 8, self.V, self.N).astype(np.int32) for _ in range(2))
        self.tok.put(tok)
        self.tgt.put(tgt)
        w = rng.standard_normal((self.V, self.D)).astype(np.float32)
        raw = bf16_bits(w) if self.dtype == "bf16" else w
        _lib.check(_lib.load().mxm_memcpy_h2d(self.table.ptr, raw.ctypes.data, raw.nbytes), "h2d")
        if self.rw:
            self.rw.put(rng.uniform(0.5, 2.0, self.N).astype(np.float32))

    def run(self, rows=None):
        n = self.N if rows is None else rows
        rw = self.rw.ptr if self.rw else 0
        self.emb.forward(n, self.tok.ptr, self.table.ptr, self.h.ptr)
        self.loss.backward(n, self.h.ptr, self.table.ptr, self.tgt.ptr, dx=self.dh.ptr, dw=self.dw.ptr,
                           row_weights=rw, loss=self.per.ptr, lse=self.lse.ptr, total=self.total.ptr)
        self.emb.backward(n, self.tok.ptr, self.dh.ptr, self.dw.ptr, accumulate=True)

    def results(self):
        self.loss.synchronize()
        return [b.get() for b in (self.h, self.per, self.lse, self.total, self.dh, self.dw)]

    def close(self):
        self.loss.close()
        self.emb.close()


@pytest.mark.parametrize("N,D,V,dtype,weighted", [
    (1, 64, 300, "bf16", False), (16, 72, 500, "fp32", False), (200, 64, 1000, "bf16", True),
    (700, 136, 900, "fp32", True), (1500, 200, 2100, "bf16", False), (2100, 40, 700, "fp32", False)])
def test_captured_and_replayed(gpu_lib, N, D, V, dtype, weighted):
    """Both ends in one graph: replays on new data in the same buffers, with eager calls on
    other data between them, give the eager call's bits."""
    ends = Ends(N, D, V, dtype, 20.0, weighted=weighted)
    ends.fill(0)
    graph = Graph(gpu_lib, ends.loss.stream(), ends.run)
    for seed in (1, 2, 3):
        ends.fill(seed)
        ends.run()
        want = ends.results()
        ends.fill(seed + 10)
        ends.run(max(1, N // 2))
        other = ends.results()
        ends.fill(seed)
        graph.replay()
        got = ends.results()
        assert not np.array_equal(other[-1], want[-1])
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a, b)
    graph.close()
    ends.close()


def test_threads(gpu_lib):
    """Distinct handles, of streams of their own and of a shared one, from several threads."""
    sizes = [(300, 64, 700, "bf16"), (1100, 72, 300, "fp32"), (5, 264, 4000, "bf16"), (64, 40, 90, "fp32")]
    want, bad = [], []
    for i, s in enumerate(sizes):
        e = Ends(*s)
        e.fill(i)
        e.run()
        want.append(e.results())
        e.close()
    first = TokenEmbedding(4, 4, 4)

    def work(i, share):
        try:
            e = Ends(*sizes[i], share=share)
            for _ in range(10):
                e.fill(i)
                for _ in range(4):
                    e.run()
                for a, b in zip(e.results(), want[i]):
                    np.testing.assert_array_equal(a, b)
            e.close()
        except BaseException as err:
            bad.append(err)

    ts = [threading.Thread(target=work, args=(i % len(sizes), first if i >= len(sizes) else None))
          for i in range(2 * len(sizes))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    first.close()
    assert not bad, bad[0]


def test_stream_outlives_its_first_handle_and_destroy_waits(gpu_lib):
    e = Ends(900, 136, 2000, "bf16")
    e.fill(3)
    e.run()
    want = e.results()
    for _ in range(3):
        e.run()
    e.emb.close()  # (calls of both handles are queued)
    e.loss.close()
    for b, w in zip((e.h, e.per, e.lse, e.total, e.dh, e.dw), want):
        np.testing.assert_array_equal(b.get(), w)
    f = Ends(900, 136, 2000, "bf16")
    f.fill(3)
    f.emb.forward(f.N, f.tok.ptr, f.table.ptr, f.h.ptr)
    f.emb.close()
    f.loss.backward(f.N, f.h.ptr, f.table.ptr, f.tgt.ptr, dx=f.dh.ptr, loss=f.per.ptr)
    f.loss.synchronize()
    np.testing.assert_array_equal(f.per.get(), want[1])
    f.loss.close()


def test_rows_of_a_step_do_not_depend_on_the_others(gpu_lib):
    """A row's loss and dx (without the mean) are those of a call of its own, to the
    order of its sums."""
    D, V, N = 72, 333, 260
    rng = np.random.default_rng(0)
    x = rng.standard_normal((N, D)).astype(np.float32)
    w = rng.standard_normal((V, D)).astype(np.float32)
    t = rng.integers(0, V, N).astype(np.int32)
    dw_, loss, gx = Dev(w), Dev.out((N,)), Dev.out((N, D))
    one, gone = Dev.out((1,)), Dev.out((1, D))
    with TokenLoss(V, D, N, dtype="fp32", mean=False) as h:
        dx_, dt = Dev(x), Dev(t, "int32")
        h.backward(N, dx_.ptr, dw_.ptr, dt.ptr, dx=gx.ptr, loss=loss.ptr)
        h.synchronize()
        every, grads = loss.get(), gx.get()
        size = np.abs(w).max() * 4 * (V + 2 * D) * U32 * 8
        for n in (0, 17, N - 1):
            a, b = Dev(x[n:n + 1]), Dev(t[n:n + 1], "int32")
            h.backward(1, a.ptr, dw_.ptr, b.ptr, dx=gone.ptr, loss=one.ptr)
            h.synchronize()
            mass = np.abs(x[n]) @ np.abs(w).T
            assert abs(one.get()[0] - every[n]) <= (2 * (D + 8) * 3 + 16) * 2 * U32 * mass.max()
            assert np.max(np.abs(gone.get()[0] - grads[n])) <= size * mass.max()


def test_more_than_fits_is_refused_and_harms_nothing(gpu_lib):
    e = Ends(100, 72, 300, "bf16")
    e.fill(1)
    e.run()
    want = e.results()
    with pytest.raises(_lib.MixMoEError, match="memory"):
        TokenLoss(4_194_304, 16384, 1 << 30, dtype="fp32", share=e.emb)
    e.run()
    with pytest.raises(_lib.MixMoEError, match="memory"):
        TokenEmbedding(4_194_304, 16384, 1 << 30, share=e.emb)
    e.run()
    for a, b in zip(e.results(), want):
        np.testing.assert_array_equal(a, b)
    e.close()
