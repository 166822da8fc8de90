"""The operators of a recurrent block as cases that can be timed and compared: the gated feed-forward layer and the gated
linear recurrence that mixes along the sequence.

``ffn``   ``gated_ffn.gated_ffn``: both projections, the activation, their product and the projection down, with the gradients of
          the input and of the three weights (``train``), or the output alone.
``scan``  ``gated_scan.gated_scan``: the recurrence's states and the last one, with the gradients of gates, values and initial state
          (``train``), or the states alone; packed sequences (``reset``), padded batches (``padded``), gates and values that are halves of
          one projection's output (``joint``).
"""
from __future__ import annotations

import math

import torch

own = False                                       # true: the framework's kernels, false: the plain forms

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _ffn(name, dtype, N, d, F, train=True, activation="silu"):
    c = {"kind": "ffn", "dtype": dtype, "N": N, "d": d, "F": F, "train": train, "activation": activation}
    return {"name": name, **c} if name else c


def _scan(name, dtype, B, T, D, train=True, activation="none", reset=0.0, padded=False, joint=False):
    c = {"kind": "scan", "dtype": dtype, "B": B, "T": T, "D": D, "train": train, "activation": activation, "reset": reset,
         "padded": padded, "joint": joint}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the tokens of one decoding step of the 124M model: one pass over the layer's weights, latency
        _ffn("ffn_decode", "bf16", 8, 768, 2048, train=False),
        # a block of 32 tokens for each of 8 sequences
        _ffn("ffn_block", "bf16", 256, 768, 2048, train=False),
        # a small model trained without autocast
        _ffn("ffn_fp32", "fp32", 1000, 384, 1024),
        # half precision, no size a multiple of a tile
        _ffn("ffn_ragged", "fp16", 4100, 1000, 2667, activation="gelu"),
        # the 124M model's layer at a per-GPU batch of 16 x 1024 tokens
        _ffn("ffn_micro", "bf16", 16384, 768, 2048),
        # the same at the whole-model configuration's global batch, 64 x 1024 tokens on one GPU
        _ffn("ffn_global", "bf16", 65536, 768, 2048),
        # one token for each of 64 sequences: the state goes one step on
        _scan("scan_decode", "bf16", 64, 1, 768, train=False),
        # packed sequences in half precision, odd sizes, gates and values from one projection
        _scan("scan_packed", "fp16", 3, 1001, 333, activation="positive", reset=0.01, joint=True),
        # a padded batch of a small model trained without autocast
        _scan("scan_fp32", "fp32", 8, 600, 384, activation="positive", padded=True),
        # 16 x 1024 tokens at the 124M model's width
        _scan("scan_micro", "bf16", 16, 1024, 768, joint=True),
        # 64 x 1024 tokens
        _scan("scan_global", "bf16", 64, 1024, 768),
        # one long sequence
        _scan("scan_long", "bf16", 1, 131072, 1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("ffn", "scan"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    train = rng.random() < 0.75
    if kind == "ffn":
        while True:
            N, d, F = _log(rng, 1, 65536), _log(rng, 32, 4096), _log(rng, 32, 12288)
            if rng.random() < 0.7:
                d, F = d - d % 8, F - F % 8
            if N * d * F <= 65536 * 768 * 2048 // (8 if dtype == "fp32" else 2) and d * F <= 1 << 25:
                break
        # (relu's slope jumps at zero: where two float32 sums of a gate have different signs, one of its gradients is another value altogether)
        return _ffn("", dtype, N, d, F, train=train, activation=rng.choice(("silu", "silu", "gelu", "gelu" if dtype == "fp32" else "relu")))
    while True:
        B, T, D = _log(rng, 1, 64), _log(rng, 1, 131072), _log(rng, 16, 4096)
        D -= D % 8 if rng.random() < 0.7 else 0
        if B * T * D <= 131072 * 1024 // (2 if dtype == "fp32" else 1):
            break
    return _scan("", dtype, B, T, D, train=train, activation=rng.choice(("none", "positive")), reset=rng.choice((0.0, 0.0, 0.003, 0.05)),
                 padded=rng.random() < 0.3, joint=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    if case["kind"] == "ffn":
        N, d, F = case["N"], case["d"], case["F"]
        # a normalised input, weights that leave gates of about one, and gradients as a scaled loss sends them
        s = {"x": normal(N, d), "w_gate": normal(F, d, std=d ** -0.5), "w_up": normal(F, d, std=d ** -0.5), "w_down": normal(d, F, std=F ** -0.5)}
        s = {k: v.requires_grad_(train) for k, v in s.items()}
        return {**case, **s, "grad": normal(N, d, std=0.01) if train else None}
    B, T, D = case["B"], case["T"], case["D"]
    # channels forget over 2 to 400 steps
    bias = -6.0 * torch.rand(D, device="cuda", generator=g)
    if case["joint"]:
        both = torch.randn(B, T, 2 * D, device="cuda", generator=g)
        both[..., :D] += bias
        both = both.to(dtype)
        gate, value = both[..., :D], both[..., D:]
    else:
        gate, value = torch.randn(B, T, D, device="cuda", generator=g).add_(bias).to(dtype), normal(B, T, D)
    state = torch.randn(B, D, device="cuda", generator=g)
    reset = lengths = None
    if case["reset"]:
        reset = torch.rand(B, T, device="cuda", generator=g) < case["reset"]
    if case["padded"]:
        lengths = torch.randint(0, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        lengths[0] = T
    s = {"gate": gate, "value": value, "state": state}
    s = {k: v.detach().requires_grad_(train) for k, v in s.items()}
    grads = (normal(B, T, D), torch.randn(B, D, device="cuda", generator=g)) if train else None
    return {**case, **s, "reset": reset, "lengths": lengths, "grads": grads}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return (_plain_ffn if state["kind"] == "ffn" else _plain_scan)(state)


def _run_own(s):
    from machinelearning_b200 import gated_ffn, gated_scan
    if s["kind"] == "ffn":
        y = gated_ffn.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=s["activation"])
        if not s["train"]:
            return {"y": y}
        dx, dg, du, dd = torch.autograd.grad(y, (s["x"], s["w_gate"], s["w_up"], s["w_down"]), s["grad"])
        return {"y": y.detach(), "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}
    h, last = gated_scan.gated_scan(s["gate"], s["value"], s["state"], activation=s["activation"], reset=s["reset"], lengths=s["lengths"])
    if not s["train"]:
        return {"h": h, "last": last}
    dg, dv, ds = torch.autograd.grad((h, last), (s["gate"], s["value"], s["state"]), s["grads"])
    return {"h": h.detach(), "last": last.detach(), "dgate": dg, "dvalue": dv, "dstate": ds}


def _activation(g, kind):
    """f(g) and f'(g)."""
    if kind == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    if kind == "gelu":
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    return g.clamp(min=0), (g > 0).to(g.dtype)


def _plain_ffn(s):
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    dtype = s["x"].dtype
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _activation(g, s["activation"])
    h = a * u
    y = (h @ wd.t()).to(dtype)
    if not s["train"]:
        return {"y": y}
    dy = s["grad"].float()
    dh = dy @ wd
    du = dh * a
    dg = dh.mul_(u).mul_(da)
    return {"y": y, "dx": (dg @ wg).add_(du @ wu).to(dtype), "dw_gate": (dg.t() @ x).to(dtype), "dw_up": (du.t() @ x).to(dtype),
            "dw_down": (dy.t() @ h).to(dtype)}


def _gates(s, to):
    """s, 1 - s and f(v), f'(v) in `to`; what stands behind a sequence's length passes the state on."""
    z, v = s["gate"].to(to), s["value"].to(to)
    p, q = torch.sigmoid(z), torch.sigmoid(-z)
    f, df = v, torch.ones_like(v)
    if s["activation"] == "positive":
        low = torch.sigmoid(v)
        f, df = torch.where(v >= 0, v + 0.5, low), torch.where(v >= 0, 1.0, low * (1 - low))
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(z.shape[1], device=z.device) < s["lengths"][:, None])[..., None]
    return p, q, f, df, live


def _affine_scan(a, b):
    """Prefixes of h -> a h + b along dimension 1, runs of 1, 2, 4, ... steps joined."""
    T, k = a.shape[1], 1
    while k < T:
        b = torch.cat((b[:, :k], torch.addcmul(b[:, k:], a[:, k:], b[:, :-k])), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return a, b


def _plain_scan(s):
    p, q, f, df, live = _gates(s, torch.float32)
    a, b = q, p * f
    if s["reset"] is not None:
        a = torch.where(s["reset"][..., None], 0.0, a)
    if live is not None:
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    h0 = s["state"][:, None]
    A, H = _affine_scan(a, b)
    h = torch.addcmul(H, A, h0)
    del A, H, b
    last, dtype = h[:, -1].clone(), s["gate"].dtype
    out = (h if live is None else torch.where(live, h, 0.0)).to(dtype)
    if not s["train"]:
        return {"h": out, "last": last}
    dh = s["grads"][0].float()
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    # from the last step to the first: G = dh + (the next step's a) (the next step's G)
    back = torch.cat((torch.ones_like(a[:, :1]), a[:, 1:].flip(1)), 1)
    A, G = _affine_scan(back, dh.flip(1))
    G = torch.addcmul(G, A, s["grads"][1][:, None]).flip(1)
    del A, back
    before = torch.cat((h0, h[:, :-1]), 1)
    if s["reset"] is not None:
        before = torch.where(s["reset"][..., None], 0.0, before)
    dz, dv = G * (f - before) * p * q, G * p * df
    if live is not None:
        dz, dv = torch.where(live, dz, 0.0), torch.where(live, dv, 0.0)
    return {"h": out, "last": last, "dgate": dz.to(dtype), "dvalue": dv.to(dtype), "dstate": a[:, 0] * G[:, 0]}


def work(case):
    size, train = DTYPES[case["dtype"]].itemsize, case["train"]
    if case["kind"] == "ffn":
        N, d, F = case["N"], case["d"], case["F"]
        once = (2 * N * d + 3 * F * d) * size
        return {"bytes": once + (2 * N * d + 3 * F * d) * size * train, "flops": 6 * N * d * F * (3 if train else 1)}
    B, T, D = case["B"], case["T"], case["D"]
    live = 0.5 * (B + 1) * T if case["padded"] else B * T     # (lengths are spread evenly, the first is T)
    # z, v and dh are read where there is a token, h, dz and dv written everywhere
    moved = (2 * live + B * T + (live + 2 * B * T) * train) * D * size + (4 if train else 2) * B * D * 4
    return {"bytes": moved + (B * T if case["reset"] else 0), "flops": (30 if train else 10) * live * D}


def exact(case, seed):
    """The same from the definitions in 64 bits: the recurrence step by step, in runs that start side by side and are joined after."""
    s = prepare(case, seed)
    f64 = torch.float64
    with torch.no_grad():
        if s["kind"] == "ffn":
            leaves = [s[k].detach().to(f64).requires_grad_(s["train"]) for k in ("x", "w_gate", "w_up", "w_down")]
            x, wg, wu, wd = leaves
            f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.nn.functional.relu}[s["activation"]]
            y = torch.empty(x.shape, dtype=f64, device="cuda")
            step = max(1, (1 << 25) // wg.shape[0])
            for i in range(0, x.shape[0], step):
                with torch.enable_grad():
                    yi = (f(x[i:i + step] @ wg.mT) * (x[i:i + step] @ wu.mT)) @ wd.mT
                y[i:i + step] = yi
                if s["train"]:
                    yi.backward(s["grad"][i:i + step].to(f64))
            out = {"y": y}
            if s["train"]:
                out.update(zip(("dx", "dw_gate", "dw_up", "dw_down"), (t.grad for t in leaves)))
            return out
        B, T, D = case["B"], case["T"], case["D"]
        run_len = max(1, int(math.sqrt(T)))
        runs = -(-T // run_len)
        z, v = s["gate"].detach().to(f64), s["value"].detach().to(f64)
        p, q = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
        f, df = v, torch.ones((), dtype=f64, device="cuda")
        if s["activation"] == "positive":
            f = torch.where(v < 0, 1 / (1 + torch.exp(-v)), v + 0.5)
            df = torch.where(v < 0, f * (1 - f), 1.0)
        live = torch.ones(B, T, 1, dtype=torch.bool, device="cuda")
        if s["lengths"] is not None:
            live = (torch.arange(T, device="cuda")[None, :, None] < s["lengths"][:, None, None])
        fresh = torch.zeros(B, T, 1, dtype=torch.bool, device="cuda") if s["reset"] is None else s["reset"][..., None] & live

        def walk(a, b, start):
            """h_t = a_t h_{t-1} + b_t, every h."""
            pad = runs * run_len - T
            a = torch.nn.functional.pad(a, (0, 0, 0, pad), value=1.0).view(B, runs, run_len, D)
            b = torch.nn.functional.pad(b, (0, 0, 0, pad)).view(B, runs, run_len, D)
            gain, end = torch.ones(B, runs, D, dtype=f64, device="cuda"), torch.zeros(B, runs, D, dtype=f64, device="cuda")
            for t in range(run_len):
                gain, end = gain * a[:, :, t], end * a[:, :, t] + b[:, :, t]
            first, h = torch.empty_like(end), start
            for r in range(runs):
                first[:, r] = h
                h = gain[:, r] * h + end[:, r]
            every = torch.empty_like(b)
            for t in range(run_len):
                first = first * a[:, :, t] + b[:, :, t]
                every[:, :, t] = first
            return every.view(B, -1, D)[:, :T]

        a = torch.where(live, torch.where(fresh, 0.0, q), 1.0)
        h0 = s["state"].detach().to(f64)
        h = walk(a, torch.where(live, p * f, 0.0), h0)
        out = {"h": torch.where(live, h, 0.0), "last": h[:, -1].clone()}
        if not s["train"]:
            return out
        dh = torch.where(live, s["grads"][0].to(f64), 0.0)
        later = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1)
        G = walk(later.flip(1), dh.flip(1), s["grads"][1].to(f64)).flip(1)
        del dh, later
        before = torch.where(fresh, 0.0, torch.cat((h0[:, None], h[:, :-1]), 1))
        return {**out, "dgate": torch.where(live, G * (f - before) * p * q, 0.0), "dvalue": torch.where(live, G * p * df, 0.0),
                "dstate": a[:, 0] * G[:, 0]}
