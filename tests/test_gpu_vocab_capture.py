"""Handles of the vocabulary's ends and captures: none is created on a stream that is being
captured, and the capture goes on."""
import ctypes

import numpy as np
import pytest

from mixlab_amd import _lib
from mixlab_amd.vocab import TokenEmbedding, TokenLoss
from oracle.vocab import embed_forward, token_loss
from tests.test_gpu_xent import inputs, tolerances
from tests.train_testutil import Dev, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [0, 1, 2])  # global, of this thread, relaxed
def test_create_within_a_capture(gpu_lib, mode):
    N, D, V = 60, 64, 90
    x, w, t = inputs(N, D, V, "fp32", 3)
    dw_, dt, out = Dev(w), Dev(t.astype(np.int32), "int32"), Dev.out((N, D))
    with TokenEmbedding(V, D, N) as e:
        stream, graph, exe = ctypes.c_void_p(e.stream()), ctypes.c_void_p(), ctypes.c_void_p()
        assert gpu_lib.hipStreamBeginCapture(stream, mode) == 0
        for make in (lambda: TokenLoss(V, D, N, dtype="fp32", share=e), lambda: TokenEmbedding(V, D, N, share=e)):
            with pytest.raises(_lib.MixMoEError, match="being captured"):
                make()
        e.forward(N, dt.ptr, dw_.ptr, out.ptr)
        assert gpu_lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert gpu_lib.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        assert gpu_lib.hipGraphDestroy(graph) == 0
        for _ in range(3):
            assert gpu_lib.hipGraphLaunch(exe, stream) == 0
            e.synchronize()
            close(out.get(), embed_forward(t, w, 1.0), 0.0, "fp32", "out")
        assert gpu_lib.hipGraphExecDestroy(exe) == 0
        # and afterwards one is
        dx_, loss = Dev(x), Dev.out((N,))
        with TokenLoss(V, D, N, dtype="fp32", share=e) as h:
            h.forward(N, dx_.ptr, dw_.ptr, dt.ptr, loss=loss.ptr)
            h.synchronize()
        ref = token_loss(x, w, t)
        close(loss.get(), ref["loss"], tolerances(x, w, ref, "fp32", 0.0, V)[0], "fp32", "loss")
