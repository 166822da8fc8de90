"""Linear cross entropy: the oracle against torch autograd in float64, the refusals, and -- on the GPU -- losses and
gradients against the oracle at the sizes, types and targets where the kernels could go wrong.

Bounds, element by element, with u half a step of the type the gradient of the logits is held in (bf16 2^-8, fp16 2^-11;
float32 is three bf16 parts: 2^-24) and u_out that of the output:

* a logit is a chain of the tensor core's additions, each off by at most a step (2^-23) of the sum of magnitudes S: after
  c = min(d, 1024) / 16 steps (float32: 256 / 16 and three parts of it) and the chunks' own additions |dl| <= e = (c + 8 + d / 256) 2^-23 S;
* a loss is the difference of a logarithm and a logit: |d loss| <= 2 e + 2^-21 (1 + |loss|) (ex2.approx is off by 2^-22, log by less);
* a probability is off by a factor exp(2 e) 2^-21: r = 2 e + 2^-20;
* dx = dl W: u on each dl (u^2 where dl is held in two parts: up to 256 rows), r on each p, the chain over V (k = V / 16, float32: 32 + V / 256) in steps of 2^-23, and the output's rounding:
  u_out |dx| + (u + k 2^-23) sum |dl w| + r sum p |w|; dw the same over the rows.  fp16: dl is held times 2^14 / max |g|, so what
  underflows is below 2^-25 2^-14 max |g| each, and outputs below the normal range are off by 2^-25.
"""
import numpy as np
import pytest
import torch

from oracle import step_f64

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0**-8, "fp16": 2.0**-11, "fp32": 2.0**-24}


def test_oracle_matches_autograd():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(23, 12, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(41, 12, generator=g, dtype=torch.float64).requires_grad_()
    t = torch.randint(0, 41, (23,), generator=g)
    t[::5] = -1
    for reduction in ("mean", "sum", "none"):
        loss = torch.nn.functional.cross_entropy(x @ w.t(), t, ignore_index=-1, reduction=reduction)
        up = torch.rand(23, generator=g, dtype=torch.float64) if reduction == "none" else None
        dx, dw = torch.autograd.grad(loss, (x, w), up)
        r = step_f64.linear_cross_entropy(x.detach().numpy(), w.detach().numpy(), t.numpy(), -1, reduction,
                                          None if up is None else up.numpy())
        assert np.abs(r["loss"] - loss.detach().numpy()).max() <= 1e-12
        assert np.abs(r["dx"] - dx.numpy()).max() <= 1e-13 and np.abs(r["dw"] - dw.numpy()).max() <= 1e-13


def test_entry_points_refuse_bad_arguments_before_any_launch():
    from machinelearning_b200 import _build, _lib
    _build.build()
    lib = _lib.load()
    tape = lambda *a: lib.nlfa_linear_ce_tape_bytes(256, *a)
    scratch = lib.nlfa_linear_ce_scratch_bytes
    assert tape(8, 100, 64, 2, 2, 2) > 0 and scratch(8, 100, 64, 2, 2, 2, 0) > 0 and scratch(8, 100, 64, 2, 2, 2, 1) > 0
    assert tape(8, 0, 64, 2, 2, 2) == 0 and tape(-1, 100, 64, 2, 2, 2) == 0 and tape(8, 100, 64, 2, 5, 2) == 0
    # a weight the products cannot read in place is copied to the tape
    assert lib.nlfa_linear_ce_tape_bytes(258, 8, 100, 64, 2, 2, 2) >= tape(8, 100, 64, 2, 2, 2) + 100 * 64 * 2
    big = 1 << 40

    def fwd(x=256, xd=2, w=256, wd=2, dt=2, t=256, tb=8, n=8, V=100, d=64, red=1, loss=256, tp=256, tpb=big, s=256, sb=big):
        return lib.nlfa_linear_ce_fwd(x, xd, w, wd, dt, t, tb, n, V, d, -1, red, loss, tp, tpb, s, sb, None)
    assert fwd(V=0) == 2 and fwd(d=0) == 2 and fwd(n=-1) == 2
    assert fwd(xd=7) == 3 and fwd(wd=-1) == 3 and fwd(dt=3) == 3
    assert fwd(tb=2) == 14 and fwd(red=3) == 14
    assert fwd(x=None) == 1 and fwd(w=None) == 1 and fwd(t=None) == 1 and fwd(loss=None) == 1 and fwd(tp=None) == 1 and fwd(s=None) == 1
    assert fwd(tp=264) == 6 and fwd(s=260) == 6
    assert fwd(x=257) == 6 and fwd(w=257) == 6 and fwd(w=258, wd=0) == 6 and fwd(t=260) == 6 and fwd(t=260, tb=4, tpb=64) == 11 and fwd(loss=258) == 6
    assert fwd(tpb=64) == 11 and fwd(sb=64) == 11

    def bwd(g=256, w=256, wd=2, xd=2, dt=2, t=256, tb=8, n=8, V=100, d=64, red=1, tp=256, tpb=big, dx=256, dw=256, s=256, sb=big):
        return lib.nlfa_linear_ce_bwd(g, w, wd, xd, dt, t, tb, n, V, d, -1, red, tp, tpb, dx, dw, s, sb, None)
    assert bwd(V=0) == 2 and bwd(wd=9) == 3 and bwd(tb=1) == 14
    assert bwd(dx=None, dw=None) == 0                            # nothing wanted
    assert bwd(g=None) == 1 and bwd(tp=None) == 1 and bwd(dx=264) == 6 and bwd(dw=264) == 6 and bwd(sb=64) == 11
    assert bwd(g=258) == 6 and bwd(w=257) == 6 and bwd(t=260) == 6 and bwd(g=None, n=0, t=None) == 1


def test_python_call_refuses_what_it_does_not_take():
    from machinelearning_b200 import head_loss
    x, w, t = torch.randn(4, 8), torch.randn(9, 8), torch.zeros(4, dtype=torch.long)
    assert not head_loss.supports(x, w, t)                       # CPU tensors
    with pytest.raises(ValueError, match="unsupported inputs"):
        head_loss.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="reduction"):
        head_loss.linear_cross_entropy(x, w, t, reduction="average")


def _inputs(dtype, n, V, d, seed=0, ignored=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, d, device="cuda", generator=g) * (2.0 / d**0.5)
    x = torch.randn(n, d, device="cuda", generator=g)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    x += (torch.rand(n, 1, device="cuda", generator=g) < 0.5) * w[t]
    if ignored:
        t[torch.rand(n, device="cuda", generator=g) < ignored] = -1
    return x.to(DT[dtype]).requires_grad_(), w.to(DT[dtype]).requires_grad_(), t


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(dtype, x, w, t, loss, dx, dw, reduction, grad=None, compute=None, dl_step=None):
    """Against the bounds of this file's head; ``compute``: what the products ran in, where it is not ``dtype``; ``dl_step``: u."""
    compute = compute or dtype
    dl_step = dl_step or HALF_STEP[compute]
    xs, ws = _np(x.to(DT[compute])), _np(w.to(DT[compute]))
    xs, ts = xs.reshape(-1, xs.shape[-1]), t.reshape(-1).cpu().numpy()
    up = None if grad is None else _np(grad).reshape(-1) if reduction == "none" else _np(grad)
    r = step_f64.linear_cross_entropy(xs, ws, ts, -1, reduction, up)
    n, d = xs.shape
    V = ws.shape[0]
    steps = 3 * 256 / 16 if compute == "fp32" else min(d, 1024) / 16
    e = (steps + 8 + d / 256) * 2.0**-23 * r["logit_sum"]
    assert np.abs(_np(loss).reshape(np.shape(r["loss"])) - r["loss"]).max() <= (2 * e + 2.0**-21 * (1 + np.abs(r["each"]).max())) * (
        max(1, (ts != -1).sum()) if reduction == "sum" else 1)
    if dx is None:
        return
    gmax = 1.0 if up is None else float(np.abs(up).max())
    if reduction == "mean":
        gmax /= max(1, (ts != -1).sum())
    for name, got, like, k in (("dx", dx, x, V), ("dw", dw, w, n)):
        want, total, prob = r[name], r[name + "_sum"], r[name + "_p"]
        got = _np(got).reshape(want.shape)
        out = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}[like.dtype]
        k = 32 + k / 256 if compute == "fp32" else k / 16
        bound = out * np.abs(want) + (dl_step + (k + 8) * 2.0**-23) * total + (2 * e + 2.0**-20) * prob
        if compute == "fp16":
            other = np.abs(ws).sum(0) if name == "dx" else np.abs(xs).sum(0)
            bound = bound + 2.0**-39 * gmax * other
        if like.dtype == torch.float16:
            bound = bound + 2.0**-25
        off = np.abs(got - want) - bound * (1 + 1e-3)            # (1e-3: products of the factors above)
        assert off.max() <= 0, (name, float(np.abs(got - want).max()), float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype,n,V,d", [
    ("bf16", 1, 1, 8), ("bf16", 1, 2, 1), ("bf16", 1, 50304, 768), ("bf16", 255, 256, 64), ("bf16", 256, 257, 72),
    ("bf16", 257, 255, 63), ("bf16", 600, 3001, 1056), ("bf16", 130, 1000, 2056), ("fp16", 3, 70, 33), ("fp16", 513, 1023, 100),
    ("fp16", 64, 511, 1500), ("fp32", 1, 3, 5), ("fp32", 300, 700, 96), ("fp32", 257, 513, 259), ("fp32", 40, 130, 1100)])
def test_loss_and_gradients(dtype, n, V, d, reduction):
    from machinelearning_b200 import head_loss
    x, w, t = _inputs(dtype, n, V, d, ignored=0.3 if n > 200 else 0.0)
    loss = head_loss.linear_cross_entropy(x, w, t, reduction=reduction)
    assert loss.dtype == torch.float32
    up = torch.rand(loss.shape, device="cuda") + 0.1 if reduction == "none" else torch.tensor(1.7, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    _check(dtype, x, w, t, loss, dx, dw, reduction, up)
    with torch.no_grad():
        assert torch.equal(head_loss.linear_cross_entropy(x, w, t, reduction=reduction), loss)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 64, 65, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_few_rows_hold_the_gradient_of_the_logits_in_two_parts(dtype, n):
    """Up to 256 rows: u is half a step of the second part (bf16 2^-16, fp16 2^-22)."""
    from machinelearning_b200 import head_loss
    x, w, t = _inputs(dtype, n, 1500, 200, seed=n)
    loss = head_loss.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    _check(dtype, x, w, t, loss, dx, dw, "sum", dl_step=HALF_STEP[dtype] ** 2)


@pytest.mark.gpu
def test_gradients_against_differences():
    """The directional derivative of the loss against its difference quotient, float32."""
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("fp32", 200, 500, 64, ignored=0.2)
    dx, dw = torch.autograd.grad(head_loss.linear_cross_entropy(x, w, t), (x, w))
    g = torch.Generator(device="cuda").manual_seed(5)
    for leaf, grad in ((x, dx), (w, dw)):
        v = torch.sign(grad) * (0.5 + torch.rand(grad.shape, device="cuda", generator=g))
        slope = float((grad.double() * v.double()).sum())
        h = 2.0**-9 / float(v.abs().max())
        with torch.no_grad():
            at = lambda s: float(head_loss.linear_cross_entropy(x + s * h * v if leaf is x else x, w + s * h * v if leaf is w else w, t))
            quotient = (at(1) - at(-1)) / (2 * h)
        # the third derivative along v, at most 2 (max |x| + max |w|)^3 per logit, enters with h^2 / 6; the losses' own 2^-21 (1 + loss)
        # over h
        assert abs(quotient - slope) <= 2e-2 * abs(slope), (quotient, slope)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,V,d", [("bf16", 24100, 25000, 64), ("fp32", 14000, 14500, 40)])
def test_vocabulary_in_pieces(dtype, n, V, d):
    """Sizes whose gradient of the logits does not fit the workspace (1 GiB): dx is summed over the pieces."""
    from machinelearning_b200 import _lib, head_loss
    lib = _lib.load()
    code = {"bf16": 2, "fp32": 0}[dtype]
    assert lib.nlfa_linear_ce_scratch_bytes(n, V, d, code, code, code, 1) < n * V * (2 if dtype == "bf16" else 6)
    x, w, t = _inputs(dtype, n, V, d, ignored=0.1)
    loss = head_loss.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    ref = torch.nn.functional.cross_entropy(x64 @ w64.t(), t, ignore_index=-1)
    rx, rw = torch.autograd.grad(ref, (x64, w64))
    # 2-norms: independent roundings of dl and of the output add up to at most 2 u; float32: see the bounds above, 2^-20 as a whole
    most = 2 * HALF_STEP[dtype] if dtype != "fp32" else 2.0**-20
    assert abs(float(loss) - float(ref)) <= 2.0**-19 * float(ref)
    for got, want in ((dx, rx), (dw, rw)):
        assert float((got.double() - want).norm() / want.norm()) <= most
    assert bool((dx[t == -1] == 0).all())


@pytest.mark.gpu
def test_rows_without_a_target_reach_nothing():
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("bf16", 700, 900, 96, ignored=0.4)
    clean = x.detach().clone()
    dirty = clean.clone()
    dirty[t == -1] = float("nan")
    dirty[t == -1, ::2] = float("inf")
    for reduction in ("mean", "none"):
        got = []
        for data in (clean, dirty):
            leaf, weight = data.clone().requires_grad_(), w.detach().clone().requires_grad_()
            loss = head_loss.linear_cross_entropy(leaf, weight, t, reduction=reduction)
            got.append((loss.detach(), *torch.autograd.grad(loss.sum(), (leaf, weight))))
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert bool((got[0][1][t == -1] == 0).all())


@pytest.mark.gpu
def test_no_target_left_and_no_rows():
    from machinelearning_b200 import head_loss
    x, w, _ = _inputs("bf16", 5, 300, 64)
    t = torch.full((5,), -1, device="cuda")
    loss = head_loss.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert torch.isnan(loss) and bool((dx == 0).all()) and bool((dw == 0).all())       # 0 / 0, as torch has it
    assert float(head_loss.linear_cross_entropy(x, w, t, reduction="sum").detach()) == 0.0
    assert bool((head_loss.linear_cross_entropy(x, w, t, reduction="none") == 0).all())
    e, te = x[:0].detach().requires_grad_(), t[:0]
    loss = head_loss.linear_cross_entropy(e, w, te, reduction="none")
    assert loss.shape == (0,)
    dx, dw = torch.autograd.grad(loss.sum(), (e, w))
    assert dx.shape == (0, 64) and bool((dw == 0).all())


@pytest.mark.gpu
def test_targets_outside_the_vocabulary_show():
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("fp16", 40, 100, 64)
    for bad in (100, 1 << 40, -7):
        t2 = t.clone()
        t2[3] = bad
        each = head_loss.linear_cross_entropy(x, w, t2, reduction="none")
        assert torch.isnan(each[3]) and int(torch.isnan(each).sum()) == 1
        dx, dw = torch.autograd.grad(head_loss.linear_cross_entropy(x, w, t2), (x, w))
        assert bool(torch.isnan(dx[3]).all()) and not bool(torch.isnan(dx[:3]).any()) and bool(torch.isnan(dw).all())


@pytest.mark.gpu
def test_logits_of_any_size():
    """Far below and above what exp takes: shifted by the maximum; a column that is -inf everywhere has no probability."""
    from machinelearning_b200 import head_loss
    x = torch.ones(3, 8, device="cuda", dtype=torch.bfloat16).requires_grad_()
    w = torch.zeros(300, 8, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = torch.linspace(-1000, -500, 300, device="cuda")
    t = torch.tensor([0, 150, 299], device="cuda")
    for shift in (0.0, 4096.0):
        ws = (w + shift).detach().requires_grad_()
        _check("bf16", x, ws, t, head_loss.linear_cross_entropy(x, ws, t, reduction="none"), None, None, "none")
    w2 = w.clone()
    w2[7] = -float("inf")
    w2.requires_grad_()
    each = head_loss.linear_cross_entropy(x, w2, t, reduction="none")
    keep = [i for i in range(300) if i != 7]
    want = step_f64.linear_cross_entropy(_np(x), _np(w2)[keep], [0, 149, 298], reduction="none")["loss"]
    assert np.abs(_np(each) - want).max() <= 2.0**-12
    (dw,) = torch.autograd.grad(each.sum(), w2)
    assert bool(torch.isfinite(dw.float()).all()) and bool((dw[7] == 0).all())


@pytest.mark.gpu
def test_layouts_types_and_autocast():
    """Any leading shape, int32 targets, strided and misaligned tensors; under autocast the products run in its type and the
    gradients come in the leaves'."""
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("bf16", 60, 333, 72)
    want = head_loss.linear_cross_entropy(x, w, t)
    gx, gw = torch.autograd.grad(want, (x, w))
    x3 = x.detach().view(3, 20, 72).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()
    store = torch.zeros(333 * 72 + 1, device="cuda", dtype=torch.bfloat16)
    store[1:] = w.detach().reshape(-1)
    w3 = store[1:].view(333, 72).requires_grad_()                # 2 bytes off
    assert w3.data_ptr() % 16 != 0
    loss = head_loss.linear_cross_entropy(x3, w3, t.view(3, 20).int())
    dx, dw = torch.autograd.grad(loss, (x3, w3))
    assert torch.equal(loss, want) and torch.equal(dx.reshape(60, 72), gx) and torch.equal(dw, gw)
    wt = w.detach().t().contiguous().t().requires_grad_()        # column by column
    assert torch.equal(torch.autograd.grad(head_loss.linear_cross_entropy(x, wt, t), wt)[0], gw)
    xf, wf = x.detach().float().requires_grad_(), w.detach().float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = head_loss.linear_cross_entropy(xf, wf, t)
    dx, dw = torch.autograd.grad(loss, (xf, wf))
    assert dx.dtype == dw.dtype == torch.float32 and torch.equal(loss, want)
    _check("fp32", xf, wf, t, loss, dx, dw, "mean", compute="bf16")
    with pytest.raises(ValueError, match="unsupported inputs"):
        head_loss.linear_cross_entropy(xf, w, t)                 # two types, no autocast
    with pytest.raises(ValueError, match="unsupported inputs"):
        head_loss.linear_cross_entropy(x, w, t.float())
    with pytest.raises(ValueError, match="unsupported inputs"):
        head_loss.linear_cross_entropy(x, w, t[:-1])


@pytest.mark.gpu
def test_one_gradient_only_and_no_second_derivative():
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("bf16", 300, 700, 64)
    loss = head_loss.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    fixed = w.detach()
    assert torch.equal(torch.autograd.grad(head_loss.linear_cross_entropy(x, fixed, t), x)[0], dx)
    assert torch.equal(torch.autograd.grad(head_loss.linear_cross_entropy(x.detach(), w, t), w)[0], dw)
    one = torch.autograd.grad(head_loss.linear_cross_entropy(x, w, t), w)[0]        # both record, one is asked for
    assert torch.equal(one, dw)
    up = torch.ones((), device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(head_loss.linear_cross_entropy(x, w, t), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


@pytest.mark.gpu
def test_reproducible_captured_and_on_another_stream():
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("bf16", 1500, 5000, 136, ignored=0.2)
    step = lambda: (lambda l: (l.detach(), *torch.autograd.grad(l, (x, w))))(head_loss.linear_cross_entropy(x, w, t))
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        kept = x.clone(), t.clone()
        x.mul_(0.5)
        t.copy_(torch.roll(t, 1))
    changed = step()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(changed, out))
    with torch.no_grad():
        x.copy_(kept[0])
        t.copy_(kept[1])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.gpu
def test_compiled_caller_matches_eager():
    from machinelearning_b200 import flash_cuda, head_loss
    assert flash_cuda.is_available()
    x, w, t = _inputs("bf16", 100, 400, 64)
    loss = head_loss.linear_cross_entropy(x, w, t)
    want = (loss.detach(), *torch.autograd.grad(loss, (x, w)))
    compiled = torch.compile(lambda x, w, t: head_loss.linear_cross_entropy(x, w, t), fullgraph=True)
    loss = compiled(x, w, t)
    assert all(torch.equal(a, b) for a, b in zip(want, (loss.detach(), *torch.autograd.grad(loss, (x, w)))))
