"""A smaller model from a larger one, as cases that can be timed and compared.

A case is a dict of plain values; ``kind`` names the operator:

  top      top_logits: the k largest logits of every row with their token ids, what a teacher's run keeps
  distill  distillation_loss: the divergence of a student's distribution from a teacher's over those ids, and, with
           ``train``, the gradient of the student's logits
  int4     int4_linear: a decode step's product with a weight of 4-bit codes and group scales, with a bias, a
           residual or the RMSNorm ahead of it

With ``own`` the calls are those of ``cdssm_hip``; without it the same in elementary torch operations in fp32.
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
EPS = 1e-6


def _package():
    path = os.path.join(os.getcwd(), "cayley-delta-state-space-model_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import cdssm_hip
    return cdssm_hip


def listed():
    return [
        # the candidates of a decode batch's next tokens, 64 rows over vocabulary 32000: latency
        {"name": "top_decode", "kind": "top", "T": 64, "V": 32000, "k": 50, "dtype": "bf16"},
        # a teacher's run over 4 sequences of 2048 tokens, its 32 largest of the default vocabulary kept: odd rows
        {"name": "top_teacher", "kind": "top", "T": 8192, "V": 50257, "k": 32, "dtype": "bf16"},
        # the same of an fp32 teacher, a ragged batch and a long list
        {"name": "top_fp32", "kind": "top", "T": 1999, "V": 32000, "k": 100, "dtype": "fp32"},
        # the loss of a test-sized student, as a debugging run steps it: latency and launches
        {"name": "distill_tiny", "kind": "distill", "T": 200, "V": 97, "K": 8, "dtype": "fp32", "tau": 1.0,
         "reduction": "mean", "empty": 0.0, "train": True},
        # a training step, 8 sequences of 2048 tokens, vocabulary 32000
        {"name": "distill_step", "kind": "distill", "T": 16384, "V": 32000, "K": 32, "dtype": "bf16", "tau": 2.0,
         "reduction": "mean", "empty": 0.0, "train": True},
        # a ragged padded batch over the default vocabulary, a loss for each token: odd rows, a tenth without a teacher
        {"name": "distill_ragged", "kind": "distill", "T": 4995, "V": 50257, "K": 64, "dtype": "fp32", "tau": 1.0,
         "reduction": "none", "empty": 0.1, "train": True},
        # evaluation of a student on held-out text, forward alone
        {"name": "distill_eval", "kind": "distill", "T": 8192, "V": 50257, "K": 32, "dtype": "bf16", "tau": 1.0,
         "reduction": "sum", "empty": 0.02, "train": False},
        # one token through a block's in_proj at d_model 1024: latency
        {"name": "int4_token", "kind": "int4", "M": 1, "N": 3104, "K": 1024, "g": 64, "bias": True, "residual": False,
         "norm": False},
        # an odd decode batch through the default model's in_proj with its norm, small groups
        {"name": "int4_norm", "kind": "int4", "M": 5, "N": 4992, "K": 768, "g": 32, "bias": True, "residual": False,
         "norm": True},
        # a decode batch's tied head at d_model 1024, vocabulary 32000
        {"name": "int4_head", "kind": "int4", "M": 64, "N": 32000, "K": 1024, "g": 128, "bias": False,
         "residual": False, "norm": False},
        # a wide layer's way down, added to the residual, a batch of 16
        {"name": "int4_wide", "kind": "int4", "M": 16, "N": 8192, "K": 28672, "g": 128, "bias": False,
         "residual": True, "norm": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["top", "distill", "distill", "int4", "int4"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "top":
        V = _log_int(rng, 50, 131072)
        most = (8192 * 50257 if dtype == "bf16" else 1999 * 32000) // V
        return {"kind": kind, "T": max(1, min(_log_int(rng, 1, 16384), most)), "V": V,
                "k": min(V, _log_int(rng, 1, 128)), "dtype": dtype}
    if kind == "distill":
        V = _log_int(rng, 50, 131072)
        most = (16384 * 32000 if dtype == "bf16" else 4995 * 50257) // V
        return {"kind": kind, "T": max(1, min(_log_int(rng, 1, 16384), most)), "V": V,
                "K": min(V, _log_int(rng, 1, 128)), "dtype": dtype, "tau": rng.choice([1.0, 2.0, 0.7, 4.0]),
                "reduction": rng.choice(["mean", "sum", "none"]), "empty": rng.choice([0.0, 0.1, 0.5]),
                "train": rng.random() < 0.75}
    # rows of 8 elements: what a model's widths are multiples of; the last group may be short
    K = 8 * _log_int(rng, 8, 3584)
    N = min(_log_int(rng, 16, 50257), 8192 * 28672 // K)
    extra = rng.choice(["", "bias", "residual", "norm"])
    return {"kind": kind, "M": _log_int(rng, 1, 64), "N": N, "K": K, "g": rng.choice([32, 64, 128]),
            "bias": extra in ("bias", "norm"), "residual": extra == "residual", "norm": extra == "norm"}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------

def _logits(T, V, g):
    """Rows as a head gives them: a normal bulk, and some 40 words of each row that stand out."""
    x = torch.randn(T, V, device="cuda", generator=g).mul_(2.0)
    at = torch.randint(0, V, (T, 40), device="cuda", generator=g)
    return x.scatter_add_(1, at, 10 * torch.rand(T, 40, device="cuda", generator=g))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if c["kind"] == "top":
        return {"c": c, "x": _logits(c["T"], c["V"], g).to(DTYPES[c["dtype"]])}
    if c["kind"] == "distill":
        T, V, K, dt = c["T"], c["V"], c["K"], DTYPES[c["dtype"]]
        # distinct ids in no order, their logits falling from the first on; the student agrees with some of them
        first = torch.randint(0, V, (T, 1), device="cuda", generator=g)
        ids = (first + torch.arange(K, device="cuda") * max(1, V // K)) % V
        tz = (14 + n(T, 1)) - torch.rand(T, K, device="cuda", generator=g).mul_(24.0 / K).cumsum(1)
        x = _logits(T, V, g).scatter_add_(1, ids, torch.rand(T, K, device="cuda", generator=g) * tz.clamp(min=0))
        if c["empty"]:
            tz[torch.rand(T, device="cuda", generator=g) < c["empty"]] = -math.inf
        up = n(T) / T if c["reduction"] == "none" else None
        return {"c": c, "x": x.to(dt).requires_grad_(c["train"]), "tz": tz.to(dt), "ids": ids, "up": up}
    M, N, K, gs = c["M"], c["N"], c["K"], c["g"]
    bf = torch.bfloat16
    # codes as a normal weight has them, the largest of a group near 7
    codes = n(N, K).mul_(2.6).round_().clamp_(-8, 7).to(torch.int8)
    scales = ((0.5 + torch.rand(N, -(-K // gs), device="cuda", generator=g)) / (2.6 * math.sqrt(K))).to(bf)
    s = {"c": c, "x": n(M, K).mul_(1.5).to(bf), "codes": codes, "scales": scales,
         "bias": n(N).to(bf) if c["bias"] else None, "residual": n(M, N).to(bf) if c["residual"] else None,
         "norm": (1 + 0.1 * n(K)).to(bf) if c["norm"] else None}
    if own:  # the weight as a serving program keeps it, laid out once when the model is loaded
        s["weight"] = _package().pack_int4(codes, scales, gs)
    return s


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------

def _plain_top(s):
    # a stable sort: of equal logits the lowest id comes first
    v, i = torch.sort(s["x"], dim=1, descending=True, stable=True)
    return v[:, :s["c"]["k"]].contiguous(), i[:, :s["c"]["k"]].contiguous()


def _plain_distill(s):
    c, tau = s["c"], s["c"]["tau"]
    x, tz, ids = s["x"].detach().float(), s["tz"].float(), s["ids"]
    part = tz != -math.inf
    has = part.any(1)
    tz = torch.where(has[:, None], tz, 0.0) / tau
    logp = tz - tz.amax(1, keepdim=True)
    logp = logp - torch.log(torch.exp(logp).sum(1, keepdim=True))
    p = torch.where(part, torch.exp(logp), 0.0)
    top = x.amax(1, keepdim=True)
    e = torch.exp((x - top) / tau)
    z = e.sum(1, keepdim=True)
    logq = (x.gather(1, ids) - top) / tau - torch.log(z)
    each = tau * tau * torch.where(part, p * (logp - logq), 0.0).sum(1)
    count = has.sum()
    loss = each if c["reduction"] == "none" else each.sum() / count if c["reduction"] == "mean" else each.sum()
    if not c["train"]:
        return loss
    up = s["up"] if s["up"] is not None else 1.0 / count if c["reduction"] == "mean" else torch.ones_like(each)
    up = tau * torch.where(has, up, 0.0)[:, None]
    return loss, e.mul_(up / z).scatter_add_(1, ids, -up * p).to(s["x"].dtype)


def _plain_int4(s):
    K, gs = s["c"]["K"], s["c"]["g"]
    w = s["codes"].float() * s["scales"].float().repeat_interleave(gs, 1)[:, :K]
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * s["norm"].float()
    y = x @ w.t()
    if s["bias"] is not None:
        y += s["bias"].float()
    if s["residual"] is not None:
        y += s["residual"].float()
    return y.to(s["x"].dtype)


def run(state):
    s, c = state, state["c"]
    if c["kind"] == "top":
        return _package().top_logits(s["x"], c["k"]) if own else _plain_top(s)
    if c["kind"] == "distill":
        if not own:
            return _plain_distill(s)
        loss = _package().distillation_loss(s["x"], s["tz"], s["ids"], temperature=c["tau"], reduction=c["reduction"])
        if not c["train"]:
            return loss
        return (loss.detach(), *torch.autograd.grad(loss, s["x"], s["up"]))
    if not own:
        return _plain_int4(s)
    return _package().int4_linear(s["x"], s["weight"], bias=s["bias"], residual=s["residual"], norm_weight=s["norm"],
                                  eps=EPS)


def work(case):
    c = case
    if c["kind"] == "top":
        b = BYTES[c["dtype"]]
        # every logit compared once
        return {"bytes": c["T"] * (b * c["V"] + (b + 8) * c["k"]), "flops": float(c["T"] * c["V"])}
    if c["kind"] == "distill":
        T, V, K, b = c["T"], c["V"], c["K"], BYTES[c["dtype"]]
        live = 1.0 - c["empty"]  # rows without a teacher are not read, their gradients are written
        each = 4 * T if c["reduction"] == "none" else 4
        return {"bytes": int(live * b * T * V) + (b * T * V if c["train"] else 0) + (b + 8) * T * K
                + each * (2 if c["train"] else 1),
                "flops": live * T * V * (8.0 if c["train"] else 4.0)}
    M, N, K = c["M"], c["N"], c["K"]
    extra = (N if c["bias"] else 0) + (M * N if c["residual"] else 0) + (K if c["norm"] else 0)
    return {"bytes": N * -(-K // 2) + 2 * (N * -(-K // c["g"]) + M * K + M * N + extra), "flops": 2.0 * M * N * K}


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "top":
        # one whole number for each logit, larger for a larger logit and, of equal ones, for a lower id
        bits = s["x"].float().view(torch.int32).long()
        rank = torch.where(bits < 0, -2 ** 31 - bits, bits) * 2 ** 20
        rank += 2 ** 20 - 1 - torch.arange(c["V"], device="cuda")
        at = torch.topk(rank, c["k"], dim=1).indices
        return s["x"].gather(1, at).double(), at
    if c["kind"] == "distill":
        tau, T, V = c["tau"], c["T"], c["V"]
        each = torch.zeros(T, device="cuda", dtype=torch.float64)
        has = (s["tz"] > -math.inf).any(1)
        weight = s["up"].double() if s["up"] is not None else torch.ones_like(each)
        if c["reduction"] == "mean":
            weight = weight / has.sum()
        grad = torch.zeros(T, V, device="cuda", dtype=torch.float64) if c["train"] else None
        for lo in range(0, T, 1024):
            rows = torch.arange(lo, min(T, lo + 1024), device="cuda")
            rows = rows[has[rows]]
            logq = torch.log_softmax(s["x"].detach()[rows].double() / tau, 1)
            logp = torch.log_softmax(s["tz"][rows].double() / tau, 1)
            full = torch.zeros_like(logq).scatter_(1, s["ids"][rows], logp.exp())
            each[rows] = tau ** 2 * (logp.exp() * (logp - logq.gather(1, s["ids"][rows]))).sum(1)
            if grad is not None:
                grad[rows] = (logq.exp() - full) * (tau * weight[rows, None])
        loss = each if c["reduction"] == "none" else each.sum() / has.sum() if c["reduction"] == "mean" else each.sum()
        return (loss, grad) if c["train"] else loss
    K, gs = c["K"], c["g"]
    x = s["x"].double()
    if s["norm"] is not None:
        x = x / (x.pow(2).sum(1, keepdim=True) / K + EPS).sqrt() * s["norm"].double()
    y = torch.zeros(c["M"], c["N"], device="cuda", dtype=torch.float64)
    for j in range(s["scales"].shape[1]):  # group by group
        part = slice(j * gs, min(K, (j + 1) * gs))
        y += (x[:, part] @ s["codes"][:, part].double().t()) * s["scales"][:, j].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["residual"] is not None:
        y += s["residual"].double()
    return y
