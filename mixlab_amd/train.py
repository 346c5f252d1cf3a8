"""A training step around the MoE op, on libmixmoe.

``ResidualNorm`` is what stands between a block's branch and the next block
(post norm, scale, gate, residual add, next norm) in both directions;
``GradientSet`` the global gradient norm, clipping and AdamW over a block's
tensors.  Both take device pointers (ints) and run asynchronously on a stream
that they can share with an op.  ``MoEBlockTrainer`` is one block's training
step built from them and the op.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import numpy as np

from . import _lib
from .moe import (DEFAULT_FFN_MULTIPLIER, OP_MOE_FEED_FORWARD, OP_RMSNORM, BlockSpec, Program,
                  WeightMeta, effective_moe_load_balance_loss_weight, emit_moe_ir,
                  moe_weight_shapes)
from .op import _DTYPES, MoEFeedForward

_GATES = {None: _lib.MXM_GATE_NONE, "row": _lib.MXM_GATE_ROW, "channel": _lib.MXM_GATE_CHANNEL}


def _stream_of(share) -> int:
    """The handle whose stream a new one runs on, 0: a stream of its own."""
    if share is None:
        return 0
    if not share.handle:
        raise ValueError("share is closed")
    return share.handle


class _Handle:
    """A handle of the library: its stream, waiting for it, its release."""

    _destroy = ""

    def _open(self, handle: int) -> None:
        if not handle:
            raise _lib.MixMoEError(_lib.last_error())
        self.handle = handle

    def stream(self) -> int:
        """The hipStream_t (as an int) that the calls run on."""
        out = ctypes.c_void_p()
        _lib.check(self._lib.mxm_stream(self.handle, ctypes.byref(out)), "mxm_stream")
        return out.value or 0

    def synchronize(self) -> None:
        _lib.check(self._lib.mxm_synchronize(self.handle), "mxm_synchronize")

    def close(self) -> None:
        if getattr(self, "handle", 0):
            getattr(self._lib, self._destroy)(self.handle)
            self.handle = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


class ResidualNorm(_Handle):
    """h = x + gate * branch_scale * post_scale * z, y = norm_scale * rms(h), with
    z = rms(delta) under post_norm, else delta (include/mixmoe.h has the
    formulas).  ``share`` is the object (an op, another of these) whose stream
    the calls run on.  branch=False leaves the norm alone: y of x."""

    _destroy = "mxm_resnorm_destroy"

    def __init__(self, D: int, max_rows: int, stream_dtype: str = "fp32", delta_dtype: str = "fp32",
                 out_dtype: str = "bf16", scale_dtype: str = "fp32", grad_dtype: str = "fp32",
                 eps: float = 1e-5, branch: bool = True, post_norm: bool = False, norm: bool = True,
                 gate: Optional[str] = None, gate_rows: int = 1, gate_sigmoid: bool = False,
                 backward: bool = True, share=None):
        stream_of = _stream_of(share)
        self._lib = _lib.init()
        flags = ((_lib.MXM_RESNORM_BRANCH if branch else 0)
                 | (_lib.MXM_RESNORM_POST_NORM if post_norm else 0)
                 | (_lib.MXM_RESNORM_NORM if norm else 0)
                 | (_lib.MXM_RESNORM_GATE_SIGMOID if gate_sigmoid else 0)
                 | (_lib.MXM_RESNORM_BACKWARD if backward else 0))
        vals = [D, max_rows, *(_DTYPES[t] for t in (stream_dtype, delta_dtype, out_dtype,
                                                    scale_dtype, grad_dtype)),
                flags, _GATES[gate], gate_rows]
        arr = (ctypes.c_int64 * len(vals))(*vals)
        self._open(self._lib.mxm_resnorm_create(arr, len(vals), float(eps), stream_of))

    def forward(self, rows: int, x: int, delta: int = 0, h: int = 0, y: int = 0,
                post_scale: int = 0, branch_scale: int = 0, gate: int = 0,
                norm_scale: int = 0) -> None:
        _lib.check(self._lib.mxm_resnorm_forward(
            self.handle, rows, x or None, delta or None, post_scale or None, branch_scale or None, gate or None,
            norm_scale or None, h or None, y or None), "mxm_resnorm_forward")

    def backward(self, rows: int, h: int = 0, delta: int = 0, dh: int = 0, dy: int = 0, dx: int = 0,
                 d_delta: int = 0, post_scale: int = 0, branch_scale: int = 0, gate: int = 0,
                 norm_scale: int = 0, d_post_scale: int = 0, d_branch_scale: int = 0,
                 d_gate: int = 0, d_norm_scale: int = 0) -> None:
        _lib.check(self._lib.mxm_resnorm_backward(
            self.handle, rows, h or None, delta or None, post_scale or None, branch_scale or None, gate or None,
            norm_scale or None, dh or None, dy or None, dx or None, d_delta or None, d_post_scale or None,
            d_branch_scale or None, d_gate or None, d_norm_scale or None), "mxm_resnorm_backward")


class GradientSet(_Handle):
    """The gradients of several tensors: their norm, clipping, AdamW.
    ``dtypes`` is one type for all or one per tensor; ``decay`` multiplies the
    weight decay of each tensor (default 1)."""

    _destroy = "mxm_grads_destroy"

    def __init__(self, sizes: Sequence[int], dtypes: Union[str, Sequence[str]] = "fp32",
                 decay: Optional[Sequence[float]] = None, share=None):
        stream_of = _stream_of(share)
        self._lib = _lib.init()
        n = len(sizes)
        if isinstance(dtypes, str):
            dtypes = [dtypes] * n
        if len(dtypes) != n or (decay is not None and len(decay) != n):
            raise ValueError(f"{n} sizes, {len(dtypes)} dtypes"
                             + ("" if decay is None else f", {len(decay)} decays"))
        self.n = n
        cs = (ctypes.c_int64 * max(1, n))(*[int(s) for s in sizes])
        cd = (ctypes.c_int32 * max(1, n))(*[_DTYPES[t] for t in dtypes])
        cw = None if decay is None else (ctypes.c_float * max(1, n))(*decay)
        self._open(self._lib.mxm_grads_create(cs, cd, cw, n, stream_of))

    def bind(self, grads: Sequence[int], clipped: Optional[Sequence[int]] = None,
             params: Optional[Sequence[int]] = None, m: Optional[Sequence[int]] = None,
             v: Optional[Sequence[int]] = None, params_bf16: Optional[Sequence[int]] = None) -> None:
        """Device pointers, one per tensor (see mxm_grads_bind)."""
        def arr(ptrs):
            if ptrs is None:
                return None
            if len(ptrs) != self.n:
                raise ValueError(f"{len(ptrs)} pointers for {self.n} tensors")
            return (ctypes.c_void_p * self.n)(*[p or None for p in ptrs])

        _lib.check(self._lib.mxm_grads_bind(self.handle, *(arr(p) for p in (
            grads, clipped, params, m, v, params_bf16))), "mxm_grads_bind")

    def norm(self, norm: int) -> None:
        _lib.check(self._lib.mxm_grads_norm(self.handle, norm or None), "mxm_grads_norm")

    def clip(self, max_norm: float, norm: int = 0) -> None:
        _lib.check(self._lib.mxm_grads_clip(self.handle, max_norm, norm or None), "mxm_grads_clip")

    def adamw(self, lr: float, beta1: float, beta2: float, eps: float, weight_decay: float,
              max_norm: float, step: int, norm: int = 0, skipped: int = 0) -> None:
        _lib.check(self._lib.mxm_grads_adamw(self.handle, lr, beta1, beta2, eps, weight_decay,
                                             max_norm, step or None, norm or None, skipped or None),
                   "mxm_grads_adamw")


class MoEBlockTrainer:
    """One MoE block in training: its forward (RMSNorm, op 74, optional post norm,
    moe_scale and gate, residual add), the backward of all of it, and AdamW with
    the gradients clipped by their global norm.

    fp32 masters, gradients and moments live in flat device buffers; under bf16
    compute the op and the scales read bf16 copies (gpu/ir_trainer.cpp:1395-1412
    casts every weight so).  Weights follow the block's metas
    (arch/moe.go:112-150), then ``moe_post_norm_scale`` with post_norm.  Matrices
    decay, vectors do not.  ``gate`` is None, "row" or "channel": values given to
    the forward for each group of gate_rows rows (a sequence: gate_rows=T).  All
    calls but ``update`` are asynchronous on the op's stream.  The residual stream
    and all gradients are fp32, the gate's values are what the compute is in."""

    def __init__(self, spec: BlockSpec, B: int, T: int, D: int,
                 mlp_mult: float = DEFAULT_FFN_MULTIPLIER, block_scales: bool = False,
                 post_norm: bool = False, gate: Optional[str] = None, gate_rows: int = 1,
                 gate_sigmoid: bool = False, compute_dtype: str = "fp32", beta1: float = 0.9,
                 beta2: float = 0.95, adam_eps: float = 1e-8, weight_decay: float = 0.01,
                 grad_clip: float = 1.0, flags: int = 0):
        prog = Program()
        emit_moe_ir(prog, spec, "x", 0, D, T, B, 0, mlp_mult, block_scales)
        eps = float(next(op for op in prog.ops if op.code == OP_RMSNORM).float_params[0])
        ff = next(op for op in prog.ops if op.code == OP_MOE_FEED_FORWARD)
        self.N, self.D = B * T, D
        self.bf16 = compute_dtype in ("bf16", "bfloat16")
        self.aux_weight = float(effective_moe_load_balance_loss_weight(spec))
        self.metas = moe_weight_shapes(spec, D, mlp_mult, block_scales)
        if post_norm:
            self.metas.append(WeightMeta("moe_post_norm_scale", [D], is_norm_scale=True, init_one=True))
        self.hyper = dict(beta1=beta1, beta2=beta2, eps=adam_eps, weight_decay=weight_decay,
                          max_norm=grad_clip)
        self.gate, self.gate_rows = gate, gate_rows
        self.op = MoEFeedForward.from_op(ff, compute_dtype=compute_dtype,
                                         flags=flags | _lib.MXM_FLAG_KEEP_FOR_BACKWARD)
        kept = "bf16" if self.bf16 else "fp32"
        self.entry = ResidualNorm(D, self.N, out_dtype=kept, scale_dtype=kept, eps=eps, branch=False,
                                  share=self.op)
        self.exit = ResidualNorm(D, self.N, scale_dtype=kept, eps=eps, post_norm=post_norm, norm=False,
                                 gate=gate, gate_rows=gate_rows, gate_sigmoid=gate_sigmoid,
                                 share=self.op)
        self._place()
        buf = _lib.DeviceBuffer
        esz = 2 if self.bf16 else 4
        self._xn, self._delta = buf(self.N * D * esz), buf(self.N * D * 4)
        self._d_delta, self._d_xn = buf(self.N * D * 4), buf(self.N * D * 4)
        self.aux, self.entropy, self.norm = buf(4), buf(4), buf(4)
        self.skipped = buf(4)
        self.step = buf(8)
        self.step.upload(np.zeros(1, np.int64))
        self._x = 0  # the last forward's input
        self._ready = False  # _g holds gradients that no update has taken

    def _place(self) -> None:
        """The tensors' places in the flat buffers: the expert matrices side by side
        as the op's backward writes their gradients, every other tensor at a
        multiple of 64 elements."""
        up = lambda n: (n + 63) // 64 * 64  # noqa: E731
        self._at, at = [0] * len(self.metas), 0
        sizes = [int(np.prod(m.shape)) for m in self.metas]
        experts = [i for i, m in enumerate(self.metas) if m.name.startswith("expert_")]
        for i in experts:
            self._at[i] = at
            at += sizes[i]
        for i in (i for i in range(len(sizes)) if i not in set(experts)):
            at = up(at)
            self._at[i] = at
            at += sizes[i]
        self._total = up(at)
        buf = _lib.DeviceBuffer
        self._p, self._g, self._m, self._v = (buf(self._total * 4) for _ in range(4))
        self._p16 = buf(self._total * 2) if self.bf16 else None
        zeros = np.zeros(self._total, np.float32)
        for b in (self._p, self._g, self._m, self._v):
            b.upload(zeros)
        self.grads = GradientSet(sizes, decay=[0.0 if len(m.shape) == 1 else 1.0 for m in self.metas],
                                 share=self.op)
        ptrs = lambda b, item: [b.value + o * item for o in self._at]  # noqa: E731
        self.grads.bind(ptrs(self._g, 4), params=ptrs(self._p, 4), m=ptrs(self._m, 4),
                        v=ptrs(self._v, 4),
                        params_bf16=ptrs(self._p16, 2) if self.bf16 else None)

    def _index(self, name: str) -> int:
        return next((i for i, m in enumerate(self.metas) if m.name == name), -1)

    def _weight(self, name: str) -> int:
        """The device pointer of a weight as the kernels read it, 0 if the block has none."""
        i = self._index(name)
        if i < 0:
            return 0
        return self._p16.value + 2 * self._at[i] if self.bf16 else self._p.value + 4 * self._at[i]

    def _grad(self, name: str) -> int:
        i = self._index(name)
        return 0 if i < 0 else self._g.value + 4 * self._at[i]

    def _bind(self) -> None:
        """The op's copies of its matrices from the masters (or their bf16 copies)."""
        src, item, code = ((self._p16, 2, _lib.MXM_DTYPE_BF16) if self.bf16
                           else (self._p, 4, _lib.MXM_DTYPE_F32))
        index = 1
        for i, m in enumerate(self.metas):
            if len(m.shape) == 2:
                self.op.set_input(index, (ctypes.c_void_p(src.value + item * self._at[i]), code, m.shape))
                index += 1

    def set_weights(self, weights) -> None:
        """fp32 arrays in the metas' order; the moments and the step start from zero."""
        from .workloads import bf16_bits
        if len(weights) != len(self.metas):
            raise ValueError(f"block takes {len(self.metas)} weights, got {len(weights)}")
        flat = np.zeros(self._total, np.float32)
        for m, w, at in zip(self.metas, weights, self._at):
            if list(np.shape(w)) != list(m.shape):
                raise ValueError(f"{m.name}: shape {list(np.shape(w))}, want {m.shape}")
            flat[at:at + np.size(w)] = np.asarray(w, np.float32).reshape(-1)
        self.op.synchronize()
        self._p.upload(flat)
        if self.bf16:
            self._p16.upload(bf16_bits(flat))
        zeros = np.zeros(self._total, np.float32)
        self._m.upload(zeros)
        self._v.upload(zeros)
        self.step.upload(np.zeros(1, np.int64))
        self._ready = False
        self._bind()

    def _read(self, b) -> list:
        self.op.synchronize()
        flat = b.download(np.float32, (self._total,))
        return [flat[at:at + int(np.prod(m.shape))].reshape(m.shape)
                for m, at in zip(self.metas, self._at)]

    def weights(self) -> list:
        """The fp32 masters in the metas' order."""
        return self._read(self._p)

    def gradients(self) -> list:
        """The last backward's gradients in the metas' order (not clipped)."""
        return self._read(self._g)

    def forward(self, x: int, out: int, gate: int = 0) -> None:
        """out [N, D] fp32 (not x's buffer: the backward reads x) for x [N, D] fp32.
        gate [ceil(N / gate_rows), 1 or D] is bf16 under bf16 compute, else fp32;
        the backward reads it again."""
        if x == out:
            raise ValueError("the block's training forward keeps x: out must be another buffer")
        if (gate != 0) != (self.gate is not None):
            raise ValueError("the forward takes a gate where the block has one, else none")
        self._x = 0  # (until all of it is queued)
        self.entry.forward(self.N, x, y=self._xn.value, norm_scale=self._weight("moe_norm_scale"))
        self.op.forward(self._xn.value, _lib.MXM_DTYPE_BF16 if self.bf16 else _lib.MXM_DTYPE_F32,
                        self.N, self._delta.value, self.aux.value, self.entropy.value)
        self.exit.forward(self.N, x, self._delta.value, out, gate=gate,
                          post_scale=self._weight("moe_post_norm_scale"),
                          branch_scale=self._weight("moe_scale"))
        self._x, self._gate = x, gate

    def backward(self, d_out: int, dx: int, d_gate: int = 0) -> None:
        """dx [N, D] (may be d_out) and the weights' gradients of the last forward, for
        the loss's gradient d_out [N, D] at its output and the weighted aux loss.
        d_gate, or 0, gets the gate's gradient in fp32."""
        if not self._x:
            raise _lib.MixMoEError("backward without a forward")
        self._ready = False
        self.exit.backward(self.N, delta=self._delta.value, dh=d_out, d_delta=self._d_delta.value,
                           gate=self._gate, d_gate=d_gate,
                           post_scale=self._weight("moe_post_norm_scale"),
                           branch_scale=self._weight("moe_scale"),
                           d_post_scale=self._grad("moe_post_norm_scale"),
                           d_branch_scale=self._grad("moe_scale"))
        first = next(i for i, m in enumerate(self.metas) if m.name.startswith("expert_"))
        _lib.check(_lib.load().mxm_moe_backward_kept(
            self.op.handle, self._d_delta.value, self.aux_weight, 0.0, self._d_xn.value,
            self._grad("router_w"), self._g.value + 4 * self._at[first]), "mxm_moe_backward_kept")
        self.entry.backward(self.N, self._x, dh=d_out, dy=self._d_xn.value, dx=dx,
                            norm_scale=self._weight("moe_norm_scale"),
                            d_norm_scale=self._grad("moe_norm_scale"))
        self._x, self._ready = 0, True

    def update(self, lr: float) -> bool:
        """One AdamW step on the last backward's gradients, which it uses up; the op
        gets the new weights.  False where a gradient was not finite and nothing
        changed."""
        if not self._ready:
            raise _lib.MixMoEError("update without a backward on these weights since the last update")
        self._ready = False
        h = self.hyper
        self.grads.adamw(lr, h["beta1"], h["beta2"], h["eps"], h["weight_decay"], h["max_norm"],
                         self.step.value, self.norm.value, self.skipped.value)
        self.op.synchronize()
        if self.skipped.download(np.int32, (1,))[0]:
            return False
        self._bind()
        return True

    def step_host(self, x: np.ndarray, d_out: np.ndarray, lr: float, gate: Optional[np.ndarray] = None):
        """Forward, backward and update on host arrays: a dict of out, aux (weighted),
        entropy, dx, d_gate (with a gate), norm and applied.  gate is fp32 [ceil(N /
        gate_rows), 1 or D] (axes of one more or less are the same), d_gate as it."""
        x = np.ascontiguousarray(x, np.float32)
        d_out = np.ascontiguousarray(d_out, np.float32)
        if x.shape != (self.N, self.D) or d_out.shape != x.shape:
            raise ValueError(f"x and d_out must be [{self.N}, {self.D}]")
        if (gate is not None) != (self.gate is not None):
            raise ValueError("a step takes a gate where the block has one, else none")
        if gate is not None:
            want = [-(-self.N // self.gate_rows), self.D if self.gate == "channel" else 1]
            long = lambda shape: [n for n in shape if n != 1]  # noqa: E731
            if long(np.shape(gate)) != long(want):
                raise ValueError(f"gate must be {want}, got {list(np.shape(gate))}")
        dev = _lib.DeviceBuffer
        bx, bo, bd = dev.from_array(x), dev(x.nbytes), dev.from_array(d_out)
        bg = bdg = None
        if gate is not None:
            gate = np.ascontiguousarray(gate, np.float32)
            if self.bf16:
                from .workloads import bf16_bits
                bg = dev.from_array(bf16_bits(gate))
            else:
                bg = dev.from_array(gate)
            bdg = dev(gate.nbytes)
        self.forward(bx.value, bo.value, bg.value if bg else 0)
        self.backward(bd.value, bd.value, bdg.value if bdg else 0)
        applied = self.update(lr)
        one = lambda b: float(b.download(np.float32, (1,))[0])  # noqa: E731
        got = dict(out=bo.download(np.float32, x.shape), dx=bd.download(np.float32, x.shape),
                   aux=self.aux_weight * one(self.aux), entropy=one(self.entropy),
                   norm=one(self.norm), applied=applied)
        if bdg:
            got["d_gate"] = bdg.download(np.float32, gate.shape)
        return got

    def close(self) -> None:
        for h in (self.entry, self.exit, self.grads, self.op):
            h.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
