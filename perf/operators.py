"""The two ends of a training step, as cases that can be timed and compared.

A case is a dict of plain values; ``kind`` names the operator:

  loss   linear_cross_entropy: the head's product with the vocabulary, the softmax cross entropy and, with
         ``train``, the gradients of the hidden states and of the weight
  embed  token_embedding: rows of the table by token id, scaled, and, with ``train``, the table's gradient
  clip   clip_grads: the 2-norm over all gradients of a model, and the gradients scaled by it

With ``own`` the calls are those of ``cdssm_hip.train``; without it the same in elementary torch operations in fp32.
``exact`` restates them in float64.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}
IGNORE = -100


def _ops():
    path = os.path.join(os.getcwd(), "cayley-delta-state-space-model_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from cdssm_hip import train
    return train


def listed():
    return [
        # the loss of a test-sized model, as a debugging run steps it: latency and launches
        {"name": "loss_tiny", "kind": "loss", "T": 200, "d": 128, "V": 97, "dtype": "fp32", "reduction": "mean",
         "ignored": 0.0, "train": True},
        # a training step's loss at d_model 1024, vocabulary 32000, 8 sequences of 2048 tokens
        {"name": "loss_step", "kind": "loss", "T": 16384, "d": 1024, "V": 32000, "dtype": "bf16", "reduction": "mean",
         "ignored": 0.0, "train": True},
        # the default model's head on a ragged padded batch, a loss for each token: odd vocabulary, odd token count
        {"name": "loss_ragged", "kind": "loss", "T": 9995, "d": 768, "V": 50257, "dtype": "bf16", "reduction": "none",
         "ignored": 0.1, "train": True},
        # evaluation of the default model: each token's loss on held-out text, forward alone
        {"name": "loss_eval", "kind": "loss", "T": 8192, "d": 768, "V": 50257, "dtype": "bf16", "reduction": "none",
         "ignored": 0.02, "train": False},
        # an fp32 run of a small batch, for comparison with a bf16 one
        {"name": "loss_fp32", "kind": "loss", "T": 2048, "d": 768, "V": 32000, "dtype": "fp32", "reduction": "mean",
         "ignored": 0.0, "train": True},
        # a decode batch of 64 tokens: latency
        {"name": "embed_token", "kind": "embed", "T": 64, "d": 1024, "V": 32000, "dtype": "bf16", "scaled": False,
         "padded": 0.0, "train": False},
        # a training step's embedding at d_model 1024, vocabulary 32000
        {"name": "embed_step", "kind": "embed", "T": 16384, "d": 1024, "V": 32000, "dtype": "bf16", "scaled": False,
         "padded": 0.0, "train": True},
        # the default model's embedding on a ragged padded batch, rows scaled by sqrt(d), the padding without gradient
        {"name": "embed_ragged", "kind": "embed", "T": 9995, "d": 768, "V": 50257, "dtype": "fp32", "scaled": True,
         "padded": 0.1, "train": True},
        # the gradients of a test-sized model, clipped in place: latency over many small tensors
        {"name": "clip_tiny", "kind": "clip", "layers": 2, "d": 128, "d_inner": 128, "N": 2, "V": 97, "dtype": "fp32",
         "out": "none", "bucket": False},
        # three layers of the default model in fp32, each gradient a tensor of its own, clipped in place
        {"name": "clip_layers", "kind": "clip", "layers": 3, "d": 768, "d_inner": 1536, "N": 16, "V": 50257,
         "dtype": "fp32", "out": "none", "bucket": False},
        # a 24-layer model's bf16 gradients, views of one bucket, clipped into the optimizer's fp32 gradients
        {"name": "clip_bucket", "kind": "clip", "layers": 24, "d": 1024, "d_inner": 1024, "N": 2, "V": 32000,
         "dtype": "bf16", "out": "fp32", "bucket": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "embed", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "loss":
        d = rng.choice([64, 128, 200, 320, 512, 768, 1000, 1024])
        V = _log_int(rng, 50, 50257)
        most = (16384 * 1024 * 32000 if dtype == "bf16" else 2048 * 768 * 32000) // (d * V)
        T = max(1, min(_log_int(rng, 1, 16384), most))
        return {"kind": kind, "T": T, "d": d, "V": V, "dtype": dtype, "reduction": rng.choice(["mean", "sum", "none"]),
                "ignored": rng.choice([0.0, 0.1, 0.5]), "train": rng.random() < 0.75}
    if kind == "embed":
        return {"kind": kind, "T": _log_int(rng, 1, 65536), "d": rng.choice([64, 100, 320, 768, 1000, 1024]),
                "V": _log_int(rng, 50, 50257), "dtype": dtype, "scaled": rng.random() < 0.5,
                "padded": rng.choice([0.0, 0.1]), "train": rng.random() < 0.75}
    d, bucket = rng.choice([64, 100, 128, 320, 768, 1024]), rng.random() < 0.5
    return {"kind": kind, "layers": rng.randint(1, 24 if bucket else 3), "d": d, "d_inner": 64 * rng.randint(1, 24),
            "N": rng.choice([2, 16]), "V": _log_int(rng, 50, 50257) if d <= 768 else _log_int(rng, 50, 32000),
            "dtype": dtype, "out": rng.choice(["none", "fp32"]) if dtype == "bf16" else "none", "bucket": bucket}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------

def _tokens(T, V, g):
    """Token ids with the frequencies of text: id i about as often as 1 / (i + 1)."""
    u = torch.rand(T, device="cuda", generator=g, dtype=torch.float64)
    return torch.exp(u * math.log(V + 1.0)).long().sub_(1).clamp_(0, V - 1)


def _model_shapes(c):
    """The parameter shapes of a model: per layer in_proj, conv, gate_proj, Q_proj, readout_proj, out_proj, norms, gates."""
    d, Di, N = c["d"], c["d_inner"], c["N"]
    H = Di // 64
    layer = [(3 * Di + H * N, d), (3 * Di + H * N,), (Di, 1, 4), (Di,), (H * (N + 5), Di), (H * (N + 5),), (H,),
             (Di, Di), (Di, H * N), (d, Di), (d,), (Di,), (Di,), (Di,), (H,), (1,)]
    return [(c["V"], d)] + layer * c["layers"] + [(d,)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "loss":
        # rows of unit RMS, leaning to their label's row by an amount that differs from token to token, so that
        # the labels' probabilities run from near zero to near one
        T, d, V = c["T"], c["d"], c["V"]
        w = n(V, d) / math.sqrt(d)
        y = _tokens(T, V, g)
        x = n(T, d) + 12 * torch.rand(T, 1, device="cuda", generator=g) * w[y]
        if c["ignored"]:
            y[torch.rand(T, device="cuda", generator=g) < c["ignored"]] = IGNORE
        up = n(T) / T if c["reduction"] == "none" else None
        return {"c": c, "x": x.to(dt).requires_grad_(c["train"]), "w": w.to(dt).requires_grad_(c["train"]), "y": y,
                "up": up}
    if c["kind"] == "embed":
        T, d, V = c["T"], c["d"], c["V"]
        ids = _tokens(T, V, g)
        pad = V - 1 if c["padded"] else None
        if c["padded"]:
            ids[torch.rand(T, device="cuda", generator=g) < c["padded"]] = pad
        return {"c": c, "ids": ids, "w": (n(V, d) / math.sqrt(d)).to(dt).requires_grad_(c["train"]),
                "gy": n(T, d).to(dt), "scale": math.sqrt(d) if c["scaled"] else 1.0, "pad": pad}
    shapes = _model_shapes(c)
    sizes = [math.prod(s) for s in shapes]
    # magnitudes that differ from tensor to tensor, as those of layers do
    mags = torch.exp(n(len(shapes))).tolist()
    if c["bucket"]:
        flat = torch.cat([(n(k) * m).to(dt) for k, m in zip(sizes, mags)])
        grads = [v.view(s) for v, s in zip(flat.split(sizes), shapes)]
    else:
        flat, grads = None, [(n(*s) * m).to(dt) for s, m in zip(shapes, mags)]
    out = outs = None
    if c["out"] == "fp32":
        out = torch.empty(sum(sizes), device="cuda", dtype=torch.float32)
        outs = [v.view(s) for v, s in zip(out.split(sizes), shapes)]
    return {"c": c, "grads": grads, "flat": flat, "outs": outs, "out": out, "max_norm": 1.0}


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------

def _plain_loss(s):
    c = s["c"]
    x, w, y = s["x"].detach().float(), s["w"].detach().float(), s["y"]
    valid = y != IGNORE
    at = y.clamp(min=0)[:, None]
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    z = e.sum(1, keepdim=True)
    each = torch.where(valid, (torch.log(z) + top - logits.gather(1, at))[:, 0], 0.0)
    count = valid.sum()
    loss = each if c["reduction"] == "none" else each.sum() / count if c["reduction"] == "mean" else each.sum()
    if not c["train"]:
        return loss
    up = s["up"] if s["up"] is not None else 1.0 / count if c["reduction"] == "mean" else torch.ones_like(loss)
    up = torch.where(valid, up, 0.0)[:, None]
    p = e.mul_(up / z)
    p.scatter_add_(1, at, -up)
    return loss, (p @ w).to(s["x"].dtype), (p.t() @ x).to(s["w"].dtype)


def _plain_embed(s):
    w, ids = s["w"].detach(), s["ids"]
    y = (w[ids].float() * s["scale"]).to(w.dtype)
    if not s["c"]["train"]:
        return y
    gy = s["gy"].float() * s["scale"]
    if s["pad"] is not None:
        gy = gy * (ids != s["pad"])[:, None]
    return y, torch.zeros(w.shape, device="cuda").index_add_(0, ids, gy).to(w.dtype)


def _plain_clip(s):
    grads = [s["flat"]] if s["flat"] is not None else s["grads"]
    norm = torch.cat([t.reshape(-1) for t in grads]).float().square().sum(dtype=torch.float64).sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    if s["outs"] is not None:
        outs = [s["out"]] if s["flat"] is not None else s["outs"]
        [o.copy_(t.float() * coef) for o, t in zip(outs, grads)]
    else:
        [t.copy_(t.float() * coef) for t in grads]
    return norm.float()


def run(state):
    s, c = state, state["c"]
    if c["kind"] == "loss":
        if not own:
            return _plain_loss(s)
        loss = _ops().linear_cross_entropy(s["x"], s["w"], s["y"], ignore_index=IGNORE, reduction=c["reduction"])
        if not c["train"]:
            return loss
        return (loss.detach(), *torch.autograd.grad(loss, (s["x"], s["w"]), s["up"]))
    if c["kind"] == "embed":
        if not own:
            return _plain_embed(s)
        y = _ops().token_embedding(s["ids"], s["w"], scale=s["scale"], padding_idx=s["pad"])
        return (y.detach(), *torch.autograd.grad(y, s["w"], s["gy"])) if c["train"] else y
    norm = _ops().clip_grads(s["grads"], s["max_norm"], out=s["outs"]) if own else _plain_clip(s)
    if s["outs"] is not None:
        return norm, s["out"]
    return norm, s["flat"] if s["flat"] is not None else s["grads"]


def work(case):
    c, b = case, BYTES[case["dtype"]]
    if c["kind"] == "loss":
        T, d, V = c["T"], c["d"], c["V"]
        each = 4 * T if c["reduction"] == "none" else 4
        # the product, and with gradients the two products of its backward
        return {"bytes": b * (T + V) * d * (2 if c["train"] else 1) + 8 * T + each,
                "flops": 2.0 * T * V * d * (3 if c["train"] else 1)}
    if c["kind"] == "embed":
        T, d, V = c["T"], c["d"], c["V"]
        return {"bytes": 8 * T + b * d * (min(T, V) + T + (T + V if c["train"] else 0)),
                "flops": float(T * d * (2 if c["train"] else 1))}
    n = sum(math.prod(s) for s in _model_shapes(c))
    return {"bytes": n * (b + (4 if c["out"] == "fp32" else b)), "flops": 3.0 * n}


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "loss":
        x, w, y = s["x"].detach().double(), s["w"].detach().double(), s["y"]
        keep = (y != IGNORE).double()
        weight = s["up"].double() if s["up"] is not None else torch.ones_like(keep)
        if c["reduction"] == "mean":
            weight = weight / keep.sum()
        weight = weight * keep
        each, dx, dw = torch.zeros_like(keep), torch.zeros_like(x), torch.zeros_like(w)
        for lo in range(0, c["T"], 2048):
            rows = slice(lo, min(c["T"], lo + 2048))
            logp = torch.log_softmax(x[rows] @ w.t(), 1)
            hot = torch.zeros_like(logp)
            hot[torch.arange(hot.shape[0], device="cuda"), y[rows].clamp(min=0)] = 1.0
            each[rows] = -(logp * hot).sum(1) * keep[rows]
            if c["train"]:
                diff = (logp.exp() - hot) * weight[rows, None]
                dx[rows] = diff @ w
                dw += diff.t() @ x[rows]
        loss = each if c["reduction"] == "none" else each.sum() / keep.sum() if c["reduction"] == "mean" else each.sum()
        return (loss, dx, dw) if c["train"] else loss
    if c["kind"] == "embed":
        w = s["w"].detach().double()
        y = s["scale"] * w.index_select(0, s["ids"])
        if not c["train"]:
            return y
        # the gradient by tokens in order: differences of a running sum at the tokens' bounds
        order = torch.argsort(s["ids"], stable=True)
        run_sum = torch.cat([torch.zeros(1, c["d"], device="cuda", dtype=torch.float64),
                             s["gy"].double()[order].cumsum(0)])
        ends = torch.bincount(s["ids"], minlength=c["V"]).cumsum(0)
        dw = s["scale"] * (run_sum[ends] - run_sum[torch.cat([ends.new_zeros(1), ends[:-1]])])
        if s["pad"] is not None:
            dw[s["pad"]] = 0
        return y, dw
    grads = [t.double() for t in ([s["flat"]] if s["flat"] is not None else s["grads"])]
    norm = math.sqrt(math.fsum(float(t.pow(2).sum()) for t in grads))
    scaled = [t * min(1.0, s["max_norm"] / (norm + 1e-6)) for t in grads]
    if s["outs"] is not None and s["flat"] is None:
        scaled = [torch.cat([t.reshape(-1) for t in scaled])]
    return torch.tensor(norm, dtype=torch.float64), (scaled[0] if len(scaled) == 1 else scaled)
