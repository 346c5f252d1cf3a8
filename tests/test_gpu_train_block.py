"""One block's training step as a program runs it: entry norm, op 74 with a kept
forward, exit with the residual; their backward; the gradients' norm, clipping
and AdamW; the op on the updated weights.  Against float64 restatements on the
values that the device's own steps kept (the routing is the op's)."""
import numpy as np
import pytest

import oracle
from mixlab_amd import _lib, moe
from mixlab_amd.workloads import round_bf16
from oracle import train as ot
from oracle.backward import backward64, forward64
from tests.moe_testutil import rel_l2

pytestmark = pytest.mark.gpu

# fp32: the op's gradients carry about 16 bits (planes of bf16 pairs, 2^-16
# relative and its sums); bf16: the flow's roundings, half a step 2^-8 at each
# of the projections, the hidden, the expert outputs and the gradients between
TOL = {"fp32": 1e-4, "bf16": 2e-2}


def _weights(rng, metas):
    ws = []
    for m in metas:
        w = rng.standard_normal(m.shape, dtype=np.float32)
        ws.append(1.0 + 0.1 * w if len(m.shape) == 1 else (0.2 if m.name == "router_w" else 0.05) * w)
    return ws


def _reference(ws, metas, x, d_out, K, aux_weight, etype, act, post_norm, gate, gate_rows, top_idx, bf16):
    r = round_bf16 if bf16 else (lambda a: np.asarray(a, np.float32))
    named = {m.name: r(w).astype(np.float64) for m, w in zip(metas, ws)}
    per = 2 if etype == 2 else 3
    mats = [r(w).astype(np.float64) for m, w in zip(metas, ws) if m.name.startswith("expert_")]
    experts = [mats[i:i + per] for i in range(0, len(mats), per)]
    x64, d64 = x.astype(np.float64), d_out.astype(np.float64)
    xn = ot.rms_norm(x64, named["moe_norm_scale"])
    if bf16:
        xn = r(xn.astype(np.float32)).astype(np.float64)
    f = forward64(xn, named["router_w"], experts, top_idx, etype, act, 0.0)
    post, scale = named.get("moe_post_norm_scale"), named.get("moe_scale")
    if gate is not None:
        gate = r(gate).astype(np.float64)
    out, _ = ot.resnorm_sum(x64, f["delta"], post, scale, gate, gate_rows, False, post_norm)
    e = ot.resnorm_backward(None, f["delta"], d64, None, post, scale, gate, gate_rows, False, post_norm)
    dxn, dwr, dexp = backward64(xn, named["router_w"], experts, top_idx, e["d_delta"], aux_weight, 0.0,
                                etype, act)
    b = ot.resnorm_backward(x64, None, d64, dxn, norm_scale=named["moe_norm_scale"])
    grads = {"moe_norm_scale": b["d_w"], "router_w": dwr, "moe_scale": e["d_scale"],
             "moe_post_norm_scale": e["d_post"]}
    flat = iter([g for ge in dexp for g in ge])
    ordered = [next(flat) if m.name.startswith("expert_") else grads[m.name] for m in metas]
    return dict(out=out, dx=b["dx"], aux=aux_weight * f["aux"], grads=ordered, d_gate=e.get("d_gate"))


@pytest.mark.parametrize("dtype,B,T,D,mult,E,K,expert,scales,post,gate", [
    ("fp32", 2, 33, 64, 2.0, 4, 2, "swiglu", False, False, None),
    ("fp32", 3, 20, 65, 1.5, 3, 1, "geglu", True, True, "channel"),
    ("fp32", 1, 50, 128, 1.0, 5, 2, "mlp", True, False, "row"),
    ("bf16", 2, 40, 256, 1.0, 4, 2, "swiglu", True, True, "channel"),
    ("bf16", 1, 64, 544, 0.5, 4, 2, "geglu", False, True, None),
])
def test_training_step(gpu_lib, dtype, B, T, D, mult, E, K, expert, scales, post, gate):
    from mixlab_amd.train import MoEBlockTrainer

    bf16, N = dtype == "bf16", B * T
    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": E, "top_k": K,
                                    "expert_block": {"type": expert}})
    etype, act, _ = moe.moe_expert_type_and_activation(spec)
    gate_rows = T if gate == "channel" else 1
    rng = np.random.default_rng(N + D)
    x, d_out = (rng.standard_normal((N, D), dtype=np.float32) for _ in range(2))
    g = None
    if gate:
        g = rng.standard_normal((-(-N // gate_rows), D if gate == "channel" else 1), dtype=np.float32)
    lr, tol = 1e-2, TOL[dtype]
    with MoEBlockTrainer(spec, B, T, D, mult, scales, post, gate, gate_rows, compute_dtype=dtype,
                         grad_clip=0.5, weight_decay=0.1) as tr:
        ws = _weights(rng, tr.metas)
        tr.set_weights(ws)
        state = [(np.zeros(m.shape), np.zeros(m.shape)) for m in tr.metas]
        for t in (1, 2):
            before = tr.weights()
            got = tr.step_host(x, d_out, lr, g)
            top_idx = tr.op.routing()["top_idx"].astype(np.int64)
            grads = tr.gradients()
            want = _reference(before, tr.metas, x, d_out, K, tr.aux_weight, etype, act, post, g,
                              gate_rows, top_idx, bf16)
            assert got["applied"]
            assert rel_l2(got["out"] - x, want["out"] - x) <= tol
            assert rel_l2(got["dx"], want["dx"]) <= tol
            assert abs(got["aux"] - want["aux"]) <= tol * abs(want["aux"])
            for m, a, b in zip(tr.metas, grads, want["grads"]):
                assert rel_l2(a, b) <= (4 if m.name == "router_w" else 1) * tol, m.name
            if gate:
                assert rel_l2(got["d_gate"], want["d_gate"]) <= tol
            # the update from the device's own gradients
            norm = ot.global_norm(grads)
            assert abs(got["norm"] - norm) <= 2 ** -23 * norm
            coef = ot.clip_coef(norm, 0.5)
            after = tr.weights()
            for i, m in enumerate(tr.metas):
                decay = 0.0 if len(m.shape) == 1 else 0.1
                p, mm, vv = ot.adamw(before[i], *state[i], coef * grads[i].astype(np.float64), t, lr,
                                     0.9, 0.95, 1e-8, decay)
                state[i] = (mm, vv)
                # an update of at most about lr, known to 2^-18 of it (a first moment's
                # terms cancel at most by the second step's ratio), and the weight's step
                assert np.max(np.abs(after[i] - p)) <= 2 ** -18 * lr + 2 ** -23 * np.max(np.abs(p)), m.name
            assert not np.array_equal(after[1], before[1])


def test_non_finite_step_changes_nothing(gpu_lib):
    from mixlab_amd.train import MoEBlockTrainer

    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": 4, "top_k": 2})
    rng = np.random.default_rng(1)
    x, d_out = (rng.standard_normal((16, 64), dtype=np.float32) for _ in range(2))
    with MoEBlockTrainer(spec, 1, 16, 64, 1.0) as tr:
        ws = _weights(rng, tr.metas)
        tr.set_weights(ws)
        bad = d_out.copy()
        bad[3, 7] = np.inf
        assert not tr.step_host(x, bad, 1e-2)["applied"]
        for a, b in zip(tr.weights(), ws):
            assert np.array_equal(a, np.asarray(b, np.float32))
        assert tr.step_host(x, d_out, 1e-2)["applied"]
        assert tr.step.download(np.int64, (1,))[0] == 1


def test_entry_and_op_match_the_fused_block(gpu_lib):
    """The training forward gives what the block's fused forward gives (up to the
    order of a row's sum of squares)."""
    from mixlab_amd.op import MoEBlock
    from mixlab_amd.train import MoEBlockTrainer

    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": 4, "top_k": 2})
    rng = np.random.default_rng(4)
    x = rng.standard_normal((24, 96), dtype=np.float32)
    with MoEBlockTrainer(spec, 1, 24, 96, 1.0, block_scales=True) as tr, \
            MoEBlock(spec, 1, 24, 96, 1.0, block_scales=True) as blk:
        ws = _weights(rng, tr.metas)
        tr.set_weights(ws)
        blk.set_weights(ws)
        got = tr.step_host(x, np.ones_like(x), 0.0)
        want, aux, _ = blk.forward_host(x)
    assert rel_l2(got["out"], want) <= 1e-5
    assert abs(got["aux"] - aux) <= 1e-5 * abs(aux)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N,D,scales", [(1, 96, True), (8, 256, False), (70, 160, True)])
def test_post_norm_block_serves_what_it_trained(gpu_lib, dtype, N, D, scales):
    """The inference block with a post norm, from one token on, gives the training
    forward's output on the trained weights."""
    from mixlab_amd.op import MoEBlock
    from mixlab_amd.train import MoEBlockTrainer

    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": 4, "top_k": 2})
    rng = np.random.default_rng(N)
    x, d_out = (rng.standard_normal((N, D), dtype=np.float32) for _ in range(2))
    with MoEBlockTrainer(spec, 1, N, D, 1.0, scales, post_norm=True, compute_dtype=dtype) as tr, \
            MoEBlock(spec, 1, N, D, 1.0, scales, compute_dtype=dtype, post_norm=True) as blk:
        tr.set_weights(_weights(rng, tr.metas))
        tr.step_host(x, d_out, 1e-2)
        assert [m.name for m in blk.metas] == [m.name for m in tr.metas]
        blk.set_weights(tr.weights())
        out, aux, ent = blk.forward_host(x)
        want = tr.step_host(x, d_out, 0.0)
        # (a bf16 op of few rows streams its weights: other sums of the same products)
        tol = 1e-5 if dtype == "fp32" else TOL[dtype]
        assert rel_l2(out - x, want["out"] - x) <= tol
        assert abs(aux - want["aux"]) <= tol * abs(want["aux"])
        assert abs(ent - want["entropy"]) <= tol * abs(want["entropy"])


def test_refusals(gpu_lib):
    from mixlab_amd.train import MoEBlockTrainer

    spec = moe.BlockSpec.from_dict({"type": "moe", "num_experts": 2, "top_k": 1})
    with MoEBlockTrainer(spec, 1, 8, 32, 1.0) as tr:
        with pytest.raises(ValueError, match="weights"):
            tr.set_weights([])
        x = _lib.DeviceBuffer(8 * 32 * 4)
        with pytest.raises(ValueError, match="another buffer"):
            tr.forward(x.value, x.value)
        with pytest.raises(ValueError, match="gate"):
            tr.forward(x.value, x.value + 4, gate=x.value)
        with pytest.raises(_lib.MixMoEError, match="without a forward"):
            tr.backward(x.value, x.value)
