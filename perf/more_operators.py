"""Cases for timing the operators at the vocabulary's two ends of a training
step: the token embedding (lookup with scaling, and its gradient by sorted
tokens) and the token loss (softmax cross entropy of the hidden rows against the
vocabulary's table without keeping the logits, alone or with its gradients).

Widths are those of the repository's benchmark configurations and tests; the
vocabularies are generic: 1024, 32768 and 50257, an odd one.
"""
from __future__ import annotations

import math

import torch

own = False  # set from outside: the plain forms (False) or the library's kernels

SCALE = 22.627417      # of the embedding: sqrt(512)


def _embed(call, N, D, V, table="fp32", out="fp32", grad="fp32", dtable="fp32", pad=0.0, add=False,
           name=None):
    c = dict(call=call, N=N, D=D, V=V, table=table, out=out, grad=grad, dtable=dtable, pad=pad, add=add)
    if name:
        c["name"] = name
    return c


def _loss(call, N, D, V, dtype="bf16", pad=0.0, weights=False, softcap=0.0, name=None):
    c = dict(call=call, N=N, D=D, V=V, dtype=dtype, pad=pad, weights=weights, softcap=softcap)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # eight sequences decoding: their tokens' rows into the fp32 stream
        _embed("lookup", 8, 1024, 32768, table="bf16", name="embed_decode8"),
        # the headline layer's batch
        _embed("lookup", 65536, 2048, 50257, table="bf16", name="embed_c4"),
        # the smallest example's training step (8 x 128 tokens, D 64)
        _embed("gradient", 1024, 64, 1024, name="embed_bw_tiny"),
        # the example width, padded sequences, bf16 gradients, added to the tied head's
        _embed("gradient", 4096, 544, 32768, grad="bf16", pad=0.2, add=True, name="embed_bw_d544"),
        # the headline layer's batch in training
        _embed("gradient", 65536, 2048, 50257, name="embed_bw_c4"),
        # scoring the single token of a decoding sequence
        _loss("loss", 1, 2048, 50257, name="loss_token"),
        # a prompt of odd length at the example width, capped logits
        _loss("loss", 1999, 544, 50257, softcap=30.0, name="loss_prompt_d544"),
        # evaluation of eight sequences of 2048 tokens at the headline layer's width
        _loss("loss", 16384, 2048, 50257, name="loss_c4"),
        # the smallest example's training step in fp32
        _loss("step", 1024, 64, 1024, dtype="fp32", name="step_tiny"),
        # fp32 training at D 512 (eight sequences of 256)
        _loss("step", 2048, 512, 32768, dtype="fp32", name="step_fp32"),
        # training at the example width: weights that leave the prompts out, capped logits
        _loss("step", 4096, 544, 32768, pad=0.3, weights=True, softcap=30.0, name="step_d544"),
        # training, eight sequences of 2048 tokens at the headline layer's width
        _loss("step", 16384, 2048, 50257, name="step_c4"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: 1 to 65536 rows of 64 to 2048 channels, a
    vocabulary of 256 to 65536 (odd ones among them); the loss up to the largest
    listed step."""
    types = ("fp32", "bf16")
    call = rng.choice(("lookup", "gradient", "gradient", "loss", "loss", "step", "step"))
    while True:
        D = _log_int(rng, 64, 2048)
        D = {0: D, 1: D // 8 * 8, 2: D // 64 * 64}[rng.choice((0, 1, 2, 2))]
        V = _log_int(rng, 256, 65536)
        V = {0: V, 1: V // 64 * 64}[rng.choice((0, 1))]
        N = _log_int(rng, 1, 65536)
        pad = rng.choice((0.0, 0.0, round(rng.uniform(0.05, 0.8), 2)))
        if call in ("lookup", "gradient"):
            if (N + V) * D > (65536 + 50257) * 2048:
                continue
            return _embed(call, N, D, V, rng.choice(types), rng.choice(types), rng.choice(types),
                          rng.choice(types), pad, call == "gradient" and rng.random() < 0.4)
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        most = 16384 * 2048 * 50257 / (6 if dtype == "fp32" else 1)
        if N * D * V > most:
            continue
        return _loss(call, N, D, V, dtype, pad, rng.random() < 0.4, rng.choice((0.0, 0.0, 30.0)))


def _bytes(t):
    return 2 if t == "bf16" else 4


def _dtype(t):
    return torch.bfloat16 if t == "bf16" else torch.float32


def _left_out(c):
    """Rows of padding: tokens or targets outside the vocabulary, or weights of zero."""
    return min(c["N"] - 1, int(c["pad"] * c["N"]))


def work(c):
    N, D, V = c["N"], c["D"], c["V"]
    rows = N - _left_out(c)
    if c["call"] == "lookup":
        return {"bytes": float(4 * N + min(rows, V) * D * _bytes(c["table"]) + N * D * _bytes(c["out"])),
                "flops": float(rows * D)}
    if c["call"] == "gradient":
        kept = 2 * min(rows, V) if c["add"] else V
        return {"bytes": float(4 * N + rows * D * _bytes(c["grad"]) + kept * D * _bytes(c["dtable"])),
                "flops": float(rows * D)}
    b = (rows + V) * D * _bytes(c["dtype"]) + N * (16 if c["weights"] else 12)
    if c["call"] == "loss":
        return {"bytes": float(b), "flops": 2.0 * rows * V * D}
    return {"bytes": float(b + (N + V) * D * _bytes(c["dtype"])), "flops": 6.0 * rows * V * D}


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    N, D, V = c["N"], c["D"], c["V"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    v = {}
    # token v with the weight log((v + 2) / (v + 1)), about 1 / (v + 1.5)
    u = torch.rand(N, generator=g, device="cuda", dtype=torch.float64)
    tokens = (torch.exp(u * math.log(V + 1)) - 1).int().clamp(0, V - 1)
    out = torch.randperm(N, generator=g, device="cuda")[:_left_out(c)]
    if c["call"] == "lookup":
        v["table"] = (0.05 * randn(V, D)).to(_dtype(c["table"]))
    elif c["call"] == "gradient":
        v["dy"] = (0.01 * randn(N, D)).to(_dtype(c["grad"]))
        if c["add"]:
            v["dtable"] = (0.01 * randn(V, D)).to(_dtype(c["dtable"]))
    else:
        # logits of standard deviation 2; the target's raised by 0 to 8, as a model that
        # has learnt something raises it
        w = randn(V, D) * (2.0 / math.sqrt(D))
        raised = 8.0 * torch.rand(N, 1, generator=g, device="cuda", dtype=torch.float32)
        t = w[tokens.long()]
        v["x"] = (randn(N, D) + t * (raised / (t * t).sum(dim=1, keepdim=True))).to(_dtype(c["dtype"]))
        v["w"] = w.to(_dtype(c["dtype"]))
        if c["weights"]:
            v["weights"] = 0.5 + torch.rand(N, generator=g, device="cuda", dtype=torch.float32)
            v["weights"][out] = 0.0
            out = out[:0]
    tokens[out] = -1
    v["tokens"] = tokens
    return v


_stream_owner = []  # the handle whose stream every state's handle runs on


def _handle(c):
    from mixlab_amd.vocab import TokenEmbedding, TokenLoss

    share = _stream_owner[0] if _stream_owner else None
    if c["call"] in ("lookup", "gradient"):
        h = TokenEmbedding(c["V"], c["D"], c["N"], table_dtype=c["table"], out_dtype=c["out"],
                           grad_dtype=c["grad"], table_grad_dtype=c["dtable"], scale=SCALE, share=share)
    else:
        h = TokenLoss(c["V"], c["D"], c["N"], dtype=c["dtype"], dx_dtype=c["dtype"],
                      dw_dtype=c["dtype"], softcap=c["softcap"], mean=True,
                      backward=c["call"] == "step", share=share)
    if not _stream_owner:
        _stream_owner.append(h)
    return h


def prepare(c, seed):
    st = dict(_inputs(c, seed), c=c)
    N, D, V = c["N"], c["D"], c["V"]

    def empty(*shape, dtype="fp32"):
        return torch.empty(*shape, device="cuda", dtype=_dtype(dtype))

    if c["call"] == "lookup":
        st["out"] = empty(N, D, dtype=c["out"])
    elif c["call"] == "gradient":
        if not c["add"]:
            st["dtable"] = empty(V, D, dtype=c["dtable"])
    else:
        st["loss"], st["lse"], st["total"] = empty(N), empty(N), empty(1)
        if c["call"] == "step":
            st["dx"], st["dw"] = empty(N, D, dtype=c["dtype"]), empty(V, D, dtype=c["dtype"])
    if own:
        st["handle"] = _handle(c)
    torch.cuda.synchronize()
    return st


OUTPUTS = {"lookup": ("out",), "gradient": ("dtable",), "loss": ("loss", "lse", "total"),
           "step": ("loss", "lse", "total", "dx", "dw")}


def run(st):
    c = st["c"]
    if own:
        _run_own(c, st)
        return {k: st[k] for k in OUTPUTS[c["call"]]}
    if c["call"] == "lookup":
        return _plain_lookup(c, st)
    if c["call"] == "gradient":
        return _plain_gradient(c, st)
    return _plain_loss(c, st)


def _run_own(c, st):
    h, N = st["handle"], c["N"]

    def ptr(key):
        return st[key].data_ptr() if key in st else 0

    if c["call"] == "lookup":
        h.forward(N, ptr("tokens"), ptr("table"), ptr("out"))
    elif c["call"] == "gradient":
        h.backward(N, ptr("tokens"), ptr("dy"), ptr("dtable"), accumulate=c["add"])
    elif c["call"] == "loss":
        h.forward(N, ptr("x"), ptr("w"), ptr("tokens"), row_weights=ptr("weights"), loss=ptr("loss"),
                  lse=ptr("lse"), total=ptr("total"))
    else:
        h.backward(N, ptr("x"), ptr("w"), ptr("tokens"), dx=ptr("dx"), dw=ptr("dw"),
                   row_weights=ptr("weights"), loss=ptr("loss"), lse=ptr("lse"), total=ptr("total"))


# ---- plain forms ----

def _plain_lookup(c, st):
    t = st["tokens"].long()
    rows = st["table"][t.clamp(min=0)].float() * SCALE
    return {"out": (rows * (t >= 0)[:, None]).to(_dtype(c["out"]))}


def _plain_gradient(c, st):
    t = st["tokens"].long()
    kept = (t >= 0).nonzero()[:, 0]
    d = torch.zeros(c["V"], c["D"], device="cuda")
    d.index_add_(0, t[kept], st["dy"][kept].float())
    d = d * SCALE
    if c["add"]:
        st["dtable"].copy_(st["dtable"].float() + d)
        return {"dtable": st["dtable"]}
    return {"dtable": d.to(_dtype(c["dtable"]))}


def _plain_loss(c, st):
    t = st["tokens"].long()
    weights = st["weights"] if c["weights"] else torch.ones(c["N"], device="cuda")
    weights = weights * (t >= 0)
    kept = (weights != 0).nonzero()[:, 0]
    t, weights = t[kept], weights[kept]
    x, w = st["x"][kept].float(), st["w"].float()
    z = x @ w.t()
    if c["softcap"]:
        z = c["softcap"] * torch.tanh(z / c["softcap"])
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    s = e.sum(dim=1, keepdim=True)
    lse = (torch.log(s) + top)[:, 0]
    loss = lse - z[torch.arange(t.shape[0], device="cuda"), t]
    whole = weights.double().sum()
    out = {"loss": torch.zeros(c["N"], device="cuda"), "lse": torch.zeros(c["N"], device="cuda")}
    out["loss"][kept], out["lse"][kept] = loss, lse
    out["total"] = ((weights.double() * loss.double()).sum() / whole).float().reshape(1)
    if c["call"] == "loss":
        return out
    g = (weights / whole.float())[:, None]
    e /= s
    e[torch.arange(t.shape[0], device="cuda"), t] -= 1.0
    e *= g
    if c["softcap"]:
        e *= 1.0 - (z / c["softcap"]) ** 2
    dx = torch.zeros(c["N"], c["D"], device="cuda")
    dx[kept] = e @ w
    out["dx"] = dx.to(_dtype(c["dtype"]))
    out["dw"] = (e.t() @ x).to(_dtype(c["dtype"]))
    return out


# ---- 64 bits ----

def exact(c, seed):
    v = _inputs(c, seed)
    t = v["tokens"].long()
    inside = (t >= 0) & (t < c["V"])
    if c["call"] == "lookup":
        out = torch.zeros(c["N"], c["D"], device="cuda", dtype=torch.float64)
        out[inside] = v["table"].double().index_select(0, t[inside]) * SCALE
        return {"out": out}
    if c["call"] == "gradient":
        d = v["dtable"].double() if c["add"] else torch.zeros(c["V"], c["D"], device="cuda", dtype=torch.float64)
        return {"dtable": d.index_add(0, t[inside], v["dy"].double()[inside], alpha=SCALE)}
    weights = inside.double() * (v["weights"].double() if c["weights"] else 1.0)
    whole = weights.sum()
    w = v["w"].double().requires_grad_(c["call"] == "step")
    zeros = torch.zeros(c["N"], device="cuda", dtype=torch.float64)
    out = {"loss": zeros, "lse": zeros.clone(), "total": zeros.new_zeros(1)}
    if c["call"] == "step":
        out["dx"] = zeros.new_zeros(c["N"], c["D"])
        out["dw"] = zeros.new_zeros(c["V"], c["D"])
    for at in range(0, c["N"], 4096):  # (the logits of a few thousand rows at a time)
        rows = torch.arange(at, min(at + 4096, c["N"]), device="cuda")
        rows = rows[weights[rows] != 0]
        x = v["x"][rows].double().requires_grad_(c["call"] == "step")
        logits = torch.matmul(x, w.transpose(0, 1))
        if c["softcap"]:
            logits = torch.tanh(logits / c["softcap"]) * c["softcap"]
        lse = torch.logsumexp(logits, dim=-1)
        loss = lse - logits.gather(1, t[rows][:, None]).squeeze(1)
        part = torch.dot(weights[rows], loss) / whole
        out["loss"][rows], out["lse"][rows] = loss.detach(), lse.detach()
        out["total"] += part.detach()
        if c["call"] == "step":
            dx, dw = torch.autograd.grad(part, (x, w))
            out["dx"][rows] = dx
            out["dw"] += dw
        del logits, lse, loss, part, x
    return out
