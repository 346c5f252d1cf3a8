"""What the block's trainer refuses before it touches the device (CPU)."""
from __future__ import annotations

import numpy as np
import pytest

from mixlab_amd.train import MoEBlockTrainer


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
