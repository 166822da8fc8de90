"""The ends of a training step as cases that can be timed and compared: the head with its loss, the token embedding,
the clip of the gradients.

``loss``   ``head_loss.linear_cross_entropy``: logits of a large vocabulary, their softmax and the cross entropy, with
           the gradients of hidden states and weight (``train``), or the losses alone (scoring).
``embed``  ``token_embedding.embedding``: scaled rows of the table, with the table's gradient (``train``), or the rows alone.
``clip``   ``grad_clip.clip_grad_norm_``: the norm of all gradients, and the clipped gradients in ``out`` where a case has one.
"""
from __future__ import annotations

import math

import torch

own = False                                       # true: the framework's kernels, false: the plain forms

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _loss(name, dtype, N, V, d, train=True, ignored=0.0, reduction="mean"):
    c = {"kind": "loss", "dtype": dtype, "N": N, "V": V, "d": d, "train": train, "ignored": ignored, "reduction": reduction}
    return {"name": name, **c} if name else c


def _embed(name, dtype, N, V, d, train=True, scale=1.0, padding=-1):
    c = {"kind": "embed", "dtype": dtype, "N": N, "V": V, "d": d, "train": train, "scale": scale, "padding": padding}
    return {"name": name, **c} if name else c


def _clip(name, dtype, layers, width, vocab, out="", max_norm=1.0, size=1e-3):
    c = {"kind": "clip", "dtype": dtype, "layers": layers, "width": width, "vocab": vocab, "out": out, "max_norm": max_norm,
         "size": size}
    return {"name": name, **c} if name else c


def listed():
    return [
        # log probabilities of a few given tokens: one pass over the head's weight, latency
        _loss("loss_score", "bf16", 8, 50304, 768, train=False, reduction="none"),
        # a small model trained without autocast
        _loss("loss_fp32", "fp32", 1000, 5003, 384),
        # padded batch in half precision: a third of the targets are ignored, no size is a multiple of a tile
        _loss("loss_ragged", "fp16", 4100, 32003, 1000, ignored=0.35, reduction="sum"),
        # the 124M model's head at a per-GPU batch of 16 x 1024 tokens
        _loss("loss_micro", "bf16", 16384, 50304, 768),
        # the same at the whole-model configuration's global batch, 64 x 1024 tokens on one GPU
        _loss("loss_global", "bf16", 65536, 50304, 768),
        # the tokens of one decoding step
        _embed("embed_decode", "bf16", 8, 50304, 768, train=False, scale=math.sqrt(768.0)),
        # a small vocabulary with padding, rows that are not a multiple of 16 bytes
        _embed("embed_odd", "fp16", 3001, 1009, 100, scale=10.0, padding=0),
        # the 124M model's table (float32 weights, as autocast training keeps them) at 16 x 1024 tokens
        _embed("embed_micro", "fp32", 16384, 50304, 768),
        # long batch of a wider model
        _embed("embed_long", "bf16", 131072, 32003, 1024, scale=32.0),
        # a few small tensors: latency
        _clip("clip_small", "fp32", 1, 65, 101, max_norm=100.0),
        # every gradient of the 124M model; the norm stays below the limit, as it does on most steps
        _clip("clip_model", "fp32", 12, 768, 50304, max_norm=100.0),
        # 16-bit gradients clipped into the optimiser's float32 ones
        _clip("clip_mixed", "bf16", 12, 768, 50304, out="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("loss", "loss", "embed", "clip"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "loss":
        while True:
            N, V, d = _log(rng, 1, 65536), _log(rng, 500, 131072), _log(rng, 64, 4096)
            d -= d % 8 if rng.random() < 0.7 else 0
            if N * V <= 65536 * 50304 and N * V * d <= 65536 * 50304 * 768 // (8 if dtype == "fp32" else 2):
                break
        return _loss("", dtype, N, V, d, train=rng.random() < 0.75, ignored=rng.choice((0.0, 0.0, 0.1, 0.6)) if N > 64 else 0.0,
                     reduction=rng.choice(("mean", "sum", "none")))
    if kind == "embed":
        while True:
            N, V, d = _log(rng, 1, 131072), _log(rng, 100, 131072), _log(rng, 32, 4096)
            d -= d % 8 if rng.random() < 0.7 else 0
            if (N + V) * d <= (131072 + 32003) * 1024:
                break
        return _embed("", dtype, N, V, d, train=rng.random() < 0.75, scale=rng.choice((1.0, math.sqrt(d))),
                      padding=rng.choice((-1, 0, 1)))
    # gradients clipped where they lie would be within the limit from the second pass on: that is what these cases are
    out = rng.choice(("", "fp32", dtype))
    return _clip("", dtype, rng.randint(1, 12), _log(rng, 33, 768), _log(rng, 50, 50304), out=out,
                 max_norm=rng.choice((0.5, 100.0)) if out else 100.0)


def _shapes(case):
    """The tensors of a model: the table, and per layer four projections, a gated feed-forward layer, norms, a scalar."""
    w, f = case["width"], 8 * case["width"] // 3
    layer = [(w, w)] * 4 + [(f, w), (f, w), (w, f), (w,), (w,), (64,), (64,), (1,)]
    return [(case["vocab"], w)] + layer * case["layers"] + [(w,)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tokens(g, N, V):
    """Ids by Zipf's law, as text has them: the most frequent token is some 8% of all."""
    weight = 1.0 / (torch.arange(V, device="cuda", dtype=torch.float64) + 2.7)
    edge = weight.cumsum(0) / weight.sum()
    u = torch.rand(N, device="cuda", dtype=torch.float64, generator=g)
    return torch.searchsorted(edge, u).clamp_(max=V - 1)


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "clip":
        sizes = [math.prod(s) for s in _shapes(case)]
        # gradients lie in one flat buffer, 16 bytes apart, as a data-parallel step's buckets have them; tensors differ in size
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += (n + 7) // 8 * 8
        flat = torch.zeros(total, device="cuda", dtype=dtype)
        for at, n in zip(starts, sizes):
            flat[at:at + n] = torch.randn(n, device="cuda", generator=g) * (case["size"] * (1.0 + at % 5))
        out = torch.zeros(total, device="cuda", dtype=DTYPES[case["out"]]) if case["out"] else None
        parameters = []
        for at, s, n in zip(starts, _shapes(case), sizes):
            p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dtype))
            p.grad = flat[at:at + n].view(s)
            parameters.append(p)
        outs = [out[at:at + n].view(s) for at, s, n in zip(starts, _shapes(case), sizes)] if out is not None else None
        return {**case, "flat": flat, "parameters": parameters, "out_flat": out, "outs": outs}
    N, V, d = case["N"], case["V"], case["d"]
    targets = _tokens(g, N, V)
    if case["kind"] == "embed":
        weight = (torch.randn(V, d, device="cuda", generator=g) * 0.02).to(dtype).requires_grad_(case["train"])
        grad = torch.randn(N, d, device="cuda", generator=g).to(dtype) if case["train"] else None
        return {**case, "idx": targets, "weight": weight, "grad": grad}
    # logits of a model that has learnt something: spread of about 2, the target's raised for half of the tokens
    std = 2.0 / math.sqrt(d)
    weight = torch.randn(V, d, device="cuda", generator=g) * std
    x = torch.randn(N, d, device="cuda", generator=g)
    know = torch.rand(N, 1, device="cuda", generator=g) < 0.5
    x = x + know * (weight[targets] * (3.0 / math.sqrt(d) / std))
    if case["ignored"]:
        targets = torch.where(torch.rand(N, device="cuda", generator=g) < case["ignored"], -1, targets)
    grad = torch.rand(N, device="cuda", generator=g) / N if case["train"] and case["reduction"] == "none" else None
    return {**case, "x": x.to(dtype).requires_grad_(case["train"]), "weight": weight.to(dtype).requires_grad_(case["train"]),
            "targets": targets, "grad": grad}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"loss": _plain_loss, "embed": _plain_embed, "clip": _plain_clip}[state["kind"]](state)


def _run_own(state):
    from machinelearning_b200 import grad_clip, head_loss, token_embedding
    if state["kind"] == "loss":
        loss = head_loss.linear_cross_entropy(state["x"], state["weight"], state["targets"], ignore_index=-1,
                                              reduction=state["reduction"])
        if not state["train"]:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (state["x"], state["weight"]), state["grad"])
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    if state["kind"] == "embed":
        out = token_embedding.embedding(state["idx"], state["weight"], scale=state["scale"],
                                        padding_idx=state["padding"] if state["padding"] >= 0 else None)
        if not state["train"]:
            return {"out": out}
        (dw,) = torch.autograd.grad(out, (state["weight"],), state["grad"])
        return {"out": out.detach(), "dw": dw}
    norm = grad_clip.clip_grad_norm_(state["parameters"], state["max_norm"], out=state["outs"])
    return {"norm": norm, "grads": state["out_flat"] if state["outs"] is not None else state["flat"]}


def _plain_loss(s):
    x, w, t = s["x"].float(), s["weight"].float(), s["targets"]
    keep = t != -1
    t = torch.where(keep, t, 0)
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    at = logits.gather(1, t[:, None])
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    each = torch.where(keep, (top + total.log() - at)[:, 0], 0.0)
    count = keep.sum()
    loss = each if s["reduction"] == "none" else each.sum() if s["reduction"] == "sum" else each.sum() / count
    if not s["train"]:
        return {"loss": loss}
    g = s["grad"] if s["reduction"] == "none" else torch.ones_like(each) if s["reduction"] == "sum" else (1.0 / count).expand_as(each)
    p.div_(total)
    p[torch.arange(t.numel(), device=t.device), t] -= 1.0
    p.mul_(torch.where(keep, g, 0.0)[:, None])
    return {"loss": loss, "dx": (p @ w).to(s["x"].dtype), "dw": (p.t() @ x).to(s["weight"].dtype)}


def _plain_embed(s):
    w = s["weight"]
    out = (w[s["idx"]].float() * s["scale"]).to(w.dtype)
    if not s["train"]:
        return {"out": out}
    g = torch.where((s["idx"] == s["padding"])[:, None], 0.0, s["grad"].float())
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, s["idx"], g).mul_(s["scale"])
    return {"out": out, "dw": dw.to(w.dtype)}


def _plain_clip(s):
    norm = s["flat"].float().square().sum(dtype=torch.float64).sqrt().float()
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if s["outs"] is None:
        return {"norm": norm, "grads": s["flat"].mul_(c)}
    return {"norm": norm, "grads": s["out_flat"].copy_(s["flat"].float() * c)}


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        again = n * DTYPES[case["out"]].itemsize if case["out"] else 0     # (in place, the norm is below the limit)
        return {"bytes": n * size + again, "flops": 2 * n + (n if again else 0)}
    N, V, d = case["N"], case["V"], case["d"]
    if case["kind"] == "embed":
        rows = min(N, V)
        moved = N * 8 + rows * d * size + N * d * size
        if case["train"]:
            moved += N * d * size + V * d * size
        return {"bytes": moved, "flops": (2 if case["train"] else 1) * N * d}
    valid = N * (1.0 - case["ignored"])
    moved = (valid * d + V * d) * size + N * 8 + 4
    if case["train"]:
        moved += (N * d + V * d) * size
    return {"bytes": moved, "flops": (8 if case["train"] else 2) * valid * V * d}


def exact(case, seed):
    """The same from the definitions in 64 bits, rows of logits a few at a time."""
    s = prepare(case, seed)
    f64 = torch.float64
    if s["kind"] == "clip":
        norm = sum(p.grad.double().pow(2).sum() for p in s["parameters"]).sqrt()
        ratio = s["max_norm"] / (norm + 1e-6)
        return {"norm": norm, "grads": s["flat"].double() * torch.minimum(ratio, torch.ones_like(ratio))}
    N, V, d = s["N"], s["V"], s["d"]
    if s["kind"] == "embed":
        w = s["weight"].detach().double()
        out = w[s["idx"]] * s["scale"]
        if not s["train"]:
            return {"out": out}
        order = torch.argsort(s["idx"], stable=True)
        ids = s["idx"][order]
        rows = s["grad"].double()[order] * s["scale"] * (ids != s["padding"])[:, None]
        dw = torch.zeros(V, d, dtype=f64, device="cuda")
        dw.index_put_((ids,), rows, accumulate=True)
        return {"out": out, "dw": dw}
    x, w, t = s["x"].detach().double(), s["weight"].detach().double(), s["targets"]
    counted = t >= 0
    g = {"none": s["grad"], "sum": torch.ones(N, device="cuda"), "mean": torch.full((N,), 1.0, device="cuda", dtype=f64) / counted.sum()}
    g = g[s["reduction"]]
    losses = torch.zeros(N, dtype=f64, device="cuda")
    dx, dw = torch.zeros(N, d, dtype=f64, device="cuda"), torch.zeros(V, d, dtype=f64, device="cuda")
    step = max(1, (1 << 27) // V)
    for at in range(0, N, step):
        rows = torch.nonzero(counted[at:at + step])[:, 0] + at
        logits = torch.mm(x[rows], w.mT)
        log_p = logits - torch.logsumexp(logits, 1, keepdim=True)
        losses[rows] = -log_p[torch.arange(rows.numel(), device="cuda"), t[rows]]
        if s["train"]:
            dl = torch.exp(log_p)
            dl.scatter_add_(1, t[rows][:, None], torch.full((rows.numel(), 1), -1.0, dtype=f64, device="cuda"))
            dl *= g[rows].double()[:, None]
            dx[rows] = torch.mm(dl, w)
            dw.addmm_(dl.mT, x[rows])
    loss = losses if s["reduction"] == "none" else losses.sum() if s["reduction"] == "sum" else losses.sum() / counted.sum()
    return {"loss": loss, "dx": dx, "dw": dw} if s["train"] else {"loss": loss}
