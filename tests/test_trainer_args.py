"""What the block's trainer refuses before it touches the device (CPU)."""
from __future__ import annotations

import numpy as np
import pytest

from mixlab_amd import _lib
from mixlab_amd.moe import WeightMeta
from mixlab_amd.train import GradientSet, MoEBlockTrainer, ResidualNorm


def _trainer(**kw):
    """A trainer of 2 x 5 tokens and 8 channels that holds no device memory."""
    tr = object.__new__(MoEBlockTrainer)
    tr.__dict__.update(dict(N=10, D=8, gate=None, gate_rows=1, bf16=False), **kw)
    return tr


X = np.zeros((10, 8), np.float32)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("gate,gate_rows,shape", [
    ("channel", 5, (2, 1)), ("channel", 5, (1, 8)), ("channel", 5, (2, 9)), ("channel", 5, (16,)),
    ("channel", 4, (2, 8)), ("channel", 1, (2, 8)), ("row", 1, (9, 1)), ("row", 1, (2, 5)),
    ("row", 5, (2, 8)), ("row", 3, (3, 1)), ("row", 1, (10, 8)), ("row", 1, ()),
])
def test_gate_shapes(gate, gate_rows, shape, bf16):
    """The kernels read and write ceil(N / gate_rows) x (1 or D) values of the gate."""
    tr = _trainer(gate=gate, gate_rows=gate_rows, bf16=bf16)
    with pytest.raises(ValueError, match="gate must be"):
        tr.step_host(X, X, 1e-3, np.zeros(shape, np.float32))


def test_gate_where_the_block_has_one():
    with pytest.raises(ValueError, match="gate"):
        _trainer().step_host(X, X, 1e-3, np.zeros((10, 1), np.float32))
    with pytest.raises(ValueError, match="gate"):
        _trainer(gate="row").step_host(X, X, 1e-3)


class _Calls:
    """Stands in for the handles and the device: every method is noted by name."""

    def __init__(self, fail=()):
        self.names, self.fail, self.handle, self.value = [], set(fail), 1, 4096

    def __getattr__(self, name):
        def call(*a, **kw):
            self.names.append(name)
            if name in self.fail:
                raise _lib.MixMoEError(name)
            return np.zeros(1, np.int32) if name == "download" else 0
        return call


@pytest.fixture
def stub(monkeypatch):
    """A trainer on such stand-ins, and what was called."""
    calls = _Calls()
    monkeypatch.setattr(_lib, "load", lambda: calls)
    metas = [WeightMeta("expert_0_w_up", [8, 8])]
    hyper = dict(beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, max_norm=1.0)
    tr = _trainer(op=calls, entry=calls, exit=calls, grads=calls, metas=metas, _at=[0], _total=64,
                  hyper=hyper, aux_weight=0.0, _x=0, _ready=False)
    for name in ("_xn", "_delta", "_d_delta", "_d_xn", "_p", "_g", "_m", "_v", "aux", "entropy", "norm",
                 "skipped", "step"):
        setattr(tr, name, calls)
    return tr, calls


def test_update_needs_a_backward(stub):
    """An update takes the gradients of a backward that ran on the present weights, once."""
    tr, calls = stub

    def refused():
        before = calls.names.count("adamw")
        with pytest.raises(_lib.MixMoEError, match="update without a backward"):
            tr.update(1e-3)
        assert calls.names.count("adamw") == before

    def step():
        tr.forward(64, 128)
        tr.backward(64, 128)

    refused()
    step()
    assert tr.update(1e-3)
    refused()
    step()
    tr.set_weights([np.zeros((8, 8))])
    refused()
    tr.forward(64, 128)
    refused()
    tr.backward(64, 128)
    assert tr.update(1e-3)


def test_backward_after_a_failed_forward(stub):
    """The op may have kept what a forward that failed gave it: an earlier forward's
    input does not go with that."""
    tr, calls = stub
    tr.forward(64, 128)
    calls.fail = {"forward"}
    with pytest.raises(_lib.MixMoEError, match="forward"):
        tr.forward(256, 512)
    calls.fail = set()
    with pytest.raises(_lib.MixMoEError, match="backward without a forward"):
        tr.backward(64, 128)


@pytest.mark.parametrize("make", [lambda share: ResidualNorm(8, 4, share=share),
                                  lambda share: GradientSet([8], share=share)])
def test_sharing_the_stream_of_a_closed_handle(make):
    """A closed object has no stream: a new one would not be in order with anything."""
    closed = object.__new__(ResidualNorm)
    closed.handle = 0
    with pytest.raises(ValueError, match="share is closed"):
        make(closed)
