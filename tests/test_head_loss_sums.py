"""Linear cross entropy where sums are long, targets sure, or few rows left: inputs whose exact results are known, so that
what a kernel's sums lose shows beside the 16-bit roundings.

All on the GPU, under bf16 autocast with float32 leaves where a gradient's own rounding would hide it.  Steps of the tensor core: each
addition is off by at most 2^-23 of the sum of magnitudes.
"""
import pytest
import torch

from test_head_loss import DT, HALF_STEP, _check


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
