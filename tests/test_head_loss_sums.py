"""Linear cross entropy where sums are long, targets sure, or few rows left: inputs whose exact results are known, so that
what a kernel's sums lose shows beside the 16-bit roundings.

All on the GPU, under bf16 autocast with float32 leaves where a gradient's own rounding would hide it.  Steps of the tensor core: each
addition is off by at most 2^-23 of the sum of magnitudes.
"""
import pytest
import torch

from test_head_loss import DT, HALF_STEP, _check, _inputs


def _gradients(x, w, t, **kw):
    from machinelearning_b200 import head_loss
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = head_loss.linear_cross_entropy(x, w, t, **kw)
    return loss.detach(), *torch.autograd.grad(loss, (x, w))


def _bf16_values(*shape, seed=0, octaves=0):
    """Positive, of bf16's values, in float32; spread over `octaves`, so that sums do not fit a float32's digits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = 0.5 + torch.rand(*shape, device="cuda", generator=g)
    return (v * torch.exp2(-octaves * torch.rand(*shape, device="cuda", generator=g))).bfloat16().float()


# A chain is 4,096 summands, 256 steps; of the chunks' sums there is one addition each, of a tile's parts one each, half a step: 2^-24.
def _most(summands):
    return (256 + 8) * 2.0**-23 + summands / 4096 * 2.0**-24 + 256 * 2.0**-24


@pytest.mark.gpu
def test_gradient_of_the_weight_over_many_rows_of_one_sign():
    """W = 0: every probability is 2^-13 in whatever precision, and a word without targets gets 2^-13 sum_i x_i."""
    n, V, d = 65536, 8192, 768
    x, w = _bf16_values(n, d, octaves=12).requires_grad_(), torch.zeros(V, d, device="cuda", requires_grad=True)
    _, _, dw = _gradients(x, w, torch.zeros(n, dtype=torch.long, device="cuda"), reduction="sum")
    want = x.detach().double().sum(0) * 2.0**-13
    assert float(((dw[1:].double() - want) / want).abs().max()) <= _most(n)


@pytest.mark.gpu
def test_gradient_of_the_rows_over_many_words_of_one_sign():
    """x = 0: every probability is 2^-17, the target's word is 0, and a row gets 2^-17 sum_v w_v (in four pieces of the vocabulary)."""
    n, V, d = 16384, 131072, 768
    w = _bf16_values(V, d, octaves=12)
    w[5] = 0
    w.requires_grad_()
    x = torch.zeros(n, d, device="cuda", requires_grad=True)
    _, dx, _ = _gradients(x, w, torch.full((n,), 5, device="cuda"), reduction="sum")
    want = w.detach().double().sum(0) * 2.0**-17
    assert float(((dx.double() - want) / want).abs().max()) <= _most(V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,V,d", [("bf16", 200, 700, 4096), ("bf16", 200, 300, 16384), ("fp16", 70, 600, 8200), ("bf16", 40, 500, 1000)])
def test_both_passes_form_the_same_logits(dtype, n, V, d):
    """Products of one sign: a logit's sum of magnitudes is the logit (about 25), and chains of the whole row would be low by more than the
    bounds of chains of 1,024 have for it.  Rows of two parts, so that the gradient of the logits hides nothing."""
    from machinelearning_b200 import head_loss
    x = _bf16_values(n, d) / 32
    w = _bf16_values(V, d, seed=1) * (32 * 25 / d)
    x, w = x.to(DT[dtype]).requires_grad_(), w.to(DT[dtype]).requires_grad_()
    t = torch.arange(n, device="cuda") % V
    loss = head_loss.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    _check(dtype, x, w, t, loss, dx, dw, "sum", dl_step=HALF_STEP[dtype] ** 2)
    # in float32 from the same operands
    xf, wf = x.detach().float().requires_grad_(), w.detach().float().requires_grad_()
    with torch.autocast("cuda", dtype=DT[dtype]):
        loss = head_loss.linear_cross_entropy(xf, wf, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (xf, wf))
    _check("fp32", xf, wf, t, loss, dx, dw, "sum", compute=dtype, dl_step=HALF_STEP[dtype] ** 2)


MARGINS = [0.0, 1.0, 5.0, 12.0, 15.0, 17.0, 20.0, 25.0, 40.0, 60.0, -3.0, -12.0, -25.0]


def _sure(dtype, n, V, target, d=72):
    """Rows of known logits: x_0 is the margin by which the target's logit lies above the others' (w_0 is 1 for the target, -1/64, 0 or 1/64 for
    the others).  w_1 is 1 for the target alone and w_2 for the others alone, with x_1 = x_2 = 0: dx_1 is p - 1 of the target, dx_2 the others'
    sum of p."""
    w = torch.zeros(V, d, device="cuda")
    w[:, 0] = (torch.arange(V, device="cuda") % 3 - 1) / 64
    w[:, 2] = 1
    w[target, :3] = torch.tensor([1.0, 1.0, 0.0], device="cuda")
    x = torch.zeros(n, d, device="cuda")
    x[:, 0] = torch.tensor(MARGINS, device="cuda").repeat(n // len(MARGINS) + 1)[:n]
    t = torch.full((n,), target, device="cuda")
    if dtype != "fp32":
        assert torch.equal(x, x.to(DT[dtype]).float()) and torch.equal(w, w.to(DT[dtype]).float())
    return x.requires_grad_(), w.requires_grad_(), t


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,target", [(13, 1000, 0), (13, 1000, 777), (64, 300, 299), (200, 1000, 777), (200, 1, 0), (13, 1, 0), (200, 1000, 999)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_tokens_the_model_is_sure_of(dtype, n, V, target):
    """Losses and p - 1 down to 1e-26, in relative terms: exp2(z log2 e) with z rounded to half a step is off by |z| 2^-24 twice (product and
    constant), ex2 and exp by 2^-22 each, sums of 1,000 and their joining by 2^-20, the logarithm and the quotient by 2^-22.  Gradients: u^2 of two parts
    in 16 bits (u = 2^-8, 2^-11), 2^-24 in float32; in fp16 what lies below 2^-25 2^-14 is lost."""
    from machinelearning_b200 import head_loss
    x, w, t = _sure(dtype, n, V, target)
    with torch.autocast("cuda", dtype=DT[dtype], enabled=dtype != "fp32"):
        each = head_loss.linear_cross_entropy(x, w, t, reduction="none")
        total = head_loss.linear_cross_entropy(x, w, t, reduction="sum")
    (dx,) = torch.autograd.grad(total, x)
    l = x.detach().double() @ w.detach().double().t()
    others = torch.cat([l[:, :target], l[:, target + 1:]], 1)
    e = torch.exp(others - l[:, target:target + 1]).sum(1)       # (margins of up to 60: no overflow)
    loss, own = torch.log1p(e), -e / (1 + e)
    z = 2 * x.detach()[:, 0].abs().double() + 2
    off = 2 * z * 2.0**-24 + 2.0**-20 + 3 * 2.0**-22
    assert bool(((each.double() - loss).abs() <= off * loss).all())
    assert abs(float(total.detach().double() - loss.sum())) <= float((off * loss).sum() + 2.0**-24 * loss.sum())
    held = 2.0**-24 if dtype == "fp32" else HALF_STEP[dtype] ** 2
    small = 2.0**-39 * V if dtype == "fp16" else 0.0
    for got, want in ((dx[:, 1], own), (dx[:, 2], -own)):        # (sums of V equal signs: steps of 2^-23 on top)
        assert bool(((got.double() - want).abs() <= (off + held + 64 * 2.0**-23) * want.abs() + small).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 100])
@pytest.mark.parametrize("target_logit,other,rest", [
    (float("inf"), 0.0, 0.0), (-float("inf"), 0.0, 0.0), (0.0, float("inf"), 0.0), (0.0, -float("inf"), 0.0),
    (0.0, -float("inf"), -float("inf")), (-float("inf"), -float("inf"), -float("inf")), (float("nan"), 0.0, 0.0), (0.0, float("nan"), 0.0)])
def test_logits_that_are_not_finite(n, target_logit, other, rest):
    """Losses and gradients of the rows are infinite, NaN or finite where torch's are."""
    from machinelearning_b200 import head_loss
    V, d, target = 300, 8, 150
    w = torch.zeros(V, d, device="cuda", dtype=torch.bfloat16)
    w[:, 0], w[target, 0], w[7, 0] = rest, target_logit, other
    x = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    x.requires_grad_(), w.requires_grad_()
    t = torch.full((n,), target, device="cuda")
    each = head_loss.linear_cross_entropy(x, w, t, reduction="none")
    logits = w.detach()[:, 0].float().expand(n, V)               # (x W^T without 0 x inf)
    want = torch.nn.functional.cross_entropy(logits, t, reduction="none")
    assert torch.allclose(each, want, rtol=2.0**-18, atol=2.0**-18, equal_nan=True)
    (dw,) = torch.autograd.grad(each.sum(), w)
    dl = torch.softmax(logits, 1)
    dl[:, target] -= 1
    got, dl = dw[:, 0].float(), dl.sum(0)
    assert torch.equal(got.isnan(), dl.isnan()) and torch.allclose(got.nan_to_num(), dl.nan_to_num(), rtol=2.0**-7, atol=2.0**-7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("reduction,n,kept", [
    ("mean", 2000, 1), ("sum", 2000, 200), ("sum", 700, 256), ("mean", 5000, 256), ("none", 257, 257), ("none", 1024, 1024), ("none", 1025, 1000),
    ("none", 1500, 1024), ("none", 6000, 700), ("sum", 1300, 0), ("none", 64, 3)])
def test_gradients_of_few_rows_in_a_call_of_many(dtype, reduction, n, kept):
    """What counts is the rows with a target: up to 256 of them, up to 1,024 with a gradient each, hold the gradient of the logits in two parts."""
    from machinelearning_b200 import head_loss
    x, w, t = _inputs(dtype, n, 900, 136, seed=n)
    g = torch.Generator(device="cuda").manual_seed(n)
    drop = torch.randperm(n, device="cuda", generator=g)[kept:]
    t[drop] = -1
    # a few of the rows are most of the sums
    up = torch.exp2(-8 * torch.rand(n, device="cuda", generator=g)) if reduction == "none" else None
    xf, wf = x.detach().float().requires_grad_(), w.detach().float().requires_grad_()
    with torch.autocast("cuda", dtype=DT[dtype]):
        loss = head_loss.linear_cross_entropy(xf, wf, t, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (xf, wf), up)
    if kept == 0:
        assert bool((dx == 0).all()) and bool((dw == 0).all())
        return
    _check("fp32", xf, wf, t, loss, dx, dw, reduction, up, compute=dtype, dl_step=HALF_STEP[dtype] ** 2)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 90])
def test_float32_values_without_three_parts_show_as_nan(n):
    """Infinities and what rounds to one in bf16: NaN in every logit they enter, no finite number."""
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("fp32", n, 200, 24)
    for bad in (-float("inf"), float("inf"), 3.4e38):
        w2, x2 = w.detach().clone(), x.detach().clone()
        w2[7, 3], x2[2, 5] = bad, bad
        each = head_loss.linear_cross_entropy(x.detach(), w2, t, reduction="none")
        assert bool(each.isnan().all())
        leaf = x2.requires_grad_()
        each = head_loss.linear_cross_entropy(leaf, w.detach(), t, reduction="none")
        want = head_loss.linear_cross_entropy(x, w, t, reduction="none")
        assert bool(each[2].isnan()) and torch.equal(each[3:], want[3:]) and torch.equal(each[:2], want[:2])
        (dx,) = torch.autograd.grad(each.sum(), leaf)
        assert bool(dx[2].isnan().all()) and not bool(dx[:2].isnan().any()) and not bool(dx[3:].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("frozen", ["weight", "x", "none"])
def test_compiled_callers_form_the_gradients_that_are_wanted(monkeypatch, frozen):
    from machinelearning_b200 import flash_cuda, head_loss
    assert flash_cuda.is_available()
    x, w, t = _inputs("bf16", 90, 300, 64)
    x, w = x.detach().requires_grad_(frozen != "x"), w.detach().requires_grad_(frozen != "weight")
    leaves = [l for l in (x, w) if l.requires_grad]
    want = torch.autograd.grad(head_loss.linear_cross_entropy(x, w, t), leaves)
    asked, bwd = [], head_loss.bwd
    monkeypatch.setattr(head_loss, "bwd", lambda *a: (asked.append(a[-2:]), bwd(*a))[1])
    compiled = torch.compile(lambda x, w, t: head_loss.linear_cross_entropy(x, w, t), backend="aot_eager", fullgraph=True)
    got = torch.autograd.grad(compiled(x, w, t), leaves)
    assert asked == [(frozen != "x", frozen != "weight")]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,n", [("bf16", 2000), ("fp16", 1300), ("fp32", 700), ("bf16", 60)])
def test_replays_with_other_numbers_of_targets(dtype, n, reduction):
    """How many rows have a target is known on the device only: a captured call follows it, across the borders of tiles and of parts."""
    from machinelearning_b200 import head_loss
    x, w, t = _inputs(dtype, n, 1200, 200)

    def step():
        loss = head_loss.linear_cross_entropy(x, w, t, reduction=reduction)
        return loss.detach(), *torch.autograd.grad(loss.sum(), (x, w))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    full = t.clone()
    for keep in (n, 257, 256, 100, 1, 0, n):
        t.copy_(full)
        t[torch.randperm(n, device="cuda")[min(keep, n):]] = -1
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.gpu
def test_saved_tensors_that_are_moved_or_recomputed():
    from torch.utils.checkpoint import checkpoint
    from machinelearning_b200 import head_loss
    x, w, t = _inputs("bf16", 300, 700, 64)
    store = torch.zeros(700 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    store[1:] = w.detach().reshape(-1)
    off = store[1:].view(700, 64).requires_grad_()               # 2 bytes off: copied to the tape; comes back aligned
    loss = head_loss.linear_cross_entropy(x, w, t)
    want = torch.autograd.grad(loss, (x, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), want))
    for weight in (w, off):
        with torch.autograd.graph.save_on_cpu():
            loss = head_loss.linear_cross_entropy(x, weight, t)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, weight)), want))
    loss = checkpoint(lambda a, b: head_loss.linear_cross_entropy(a, b, t), x, w, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), want))
