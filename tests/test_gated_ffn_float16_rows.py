"""Gated feed-forward layer in float16: tokens of very different lengths, in x and in the gradient, do not cost one another digits.

h, dg and du carry a power of two per token: a token's y and dx are as exact as they would be without the others.  Weight gradients are sums over tokens and are as
exact as the largest token's share lets a float16 operand be: 2^-30 and less of that share, which is 2^-11 of one 10^5 times smaller.  So every element is held to the bounds that
test_gated_ffn.py has for tokens of one length, from the magnitudes and roundings of its own summands; and a token's y and dx as a whole to 1.2 u, two independent
roundings of u / sqrt(3) each, with what float16 leaves below its normal range, 2^-25 an element.
"""
import numpy as np
import pytest
import torch

from oracle import block_f64
from test_gated_ffn import HALF_STEP, NAMES, _bounds, _inputs, _np

HALF = torch.float16


def _case(n, x_times, dy_times, seed=0):
    """Token 17 has x_times its length, token 40 dy_times its gradient."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(HALF, n, 256, 512, 128, seed=seed, up=2.0**-8)
    with torch.no_grad():
        leaves[0][17] *= x_times
        dy[40] *= dy_times
    dy = dy.half()
    y = gated_ffn.gated_ffn(*leaves)
    want = block_f64.gated_ffn(*(_np(t) for t in leaves), "silu", _np(dy), step=1.0)
    return leaves, dy, (y, *torch.autograd.grad(y, leaves, dy)), want


def _check(got, want, name, hidden, rows=None):
    off, bound = np.abs(_np(got) - want[name]), _bounds(want, name, HALF, HALF, hidden)
    if rows is not None:
        off, bound = off[rows], bound[rows]
    assert (off <= bound).all(), (name, float((off / bound).max()))
    if rows is not None:
        whole, size = np.linalg.norm(off), np.linalg.norm(want[name][rows])
        assert whole <= 1.2 * 2.0**-11 * size + 2.0**-25 * off.size**0.5, (name, whole / size)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [200, 320])
@pytest.mark.parametrize("x_times,dy_times", [(1, 1), (1000, 1), (5000, 1), (100, 1000), (100, 10000), (1, 60000), (2.0**-12, 1), (1, 0)])
def test_long_tokens_and_the_others(n, x_times, dy_times):
    hidden = HALF_STEP[HALF]**2 if n <= 256 else None
    leaves, dy, (y, dx, *dw), want = _case(n, x_times, dy_times)
    # (what a long token gives may be outside float16)
    rows = np.array([i for i in range(n) if i not in (17, 40)])
    _check(y, want, "y", hidden, rows)
    _check(dx, want, "dx", hidden, rows)
    for i in (17, 40):
        if np.abs(want["y"][i]).max() < 6e4 and np.abs(want["dx"][i]).max() < 6e4:
            _check(y, want, "y", hidden, [i])
            _check(dx, want, "dx", hidden, [i])
    for name, g in zip(NAMES[1:], dw):
        if np.abs(want[name]).max() < 6e4:
            _check(g, want, name, hidden)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [200, 320])
def test_a_long_token_without_a_gradient_costs_the_weights_nothing(n):
    """20,000 times the others' length, and a gradient of zero: the weights' gradients are the others'."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(HALF, n, 256, 512, 128, up=2.0**-8)
    with torch.no_grad():
        leaves[0][17] = leaves[0][17].sign() * 20000
        dy[17] = 0
    dy = dy.half()
    grads = torch.autograd.grad(gated_ffn.gated_ffn(*leaves), leaves, dy)
    want = block_f64.gated_ffn(*(_np(t) for t in leaves), "silu", _np(dy), step=1.0)
    hidden = HALF_STEP[HALF]**2 if n <= 256 else None
    for name, g in zip(NAMES, grads):
        _check(g, want, name, hidden)


@pytest.mark.gpu
def test_a_token_does_not_depend_on_the_others():
    """y and dx of a token bit by bit, whatever another one holds."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(HALF, 300, 128, 256, 64)
    dy = dy.half()

    def run(x, dy):
        x = x.detach().requires_grad_()
        y = gated_ffn.gated_ffn(x, *leaves[1:])
        return y, torch.autograd.grad(y, x, dy)[0]
    y, dx = run(leaves[0], dy)
    others = torch.arange(300, device="cuda") != 9
    for times in (300.0, 0.0, float("inf"), float("nan")):
        x2, dy2 = leaves[0].detach().clone(), dy.clone()
        x2[9] *= times
        dy2[9] *= times
        y2, dx2 = run(x2, dy2)
        assert torch.equal(y2[others], y[others]) and torch.equal(dx2[others], dx[others])


@pytest.mark.gpu
def test_gradients_of_outputs_beside_one_that_is_not_finite():
    """One infinite element of dy: the rows of w_down's gradient that it does not enter are as without it."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(HALF, 300, 128, 256, 64)
    dy = dy.half()
    want = block_f64.gated_ffn(*(_np(t) for t in leaves), "silu", _np(dy), step=1.0)
    dy[5, 3] = float("inf")
    dwd = torch.autograd.grad(gated_ffn.gated_ffn(*leaves), leaves[3], dy)[0]
    _check(dwd, want, "dw_down", None, np.array([i for i in range(64) if i != 3]))
    assert not bool(torch.isfinite(dwd[3]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
def test_long_tokens_under_autocast(kind):
    """float32 leaves, odd widths (every operand is copied), one long token."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.float32, 270, 100, 333, 70, up=2.0**-8)
    with torch.no_grad():
        leaves[0][17] *= 3000
    dy = dy.half()
    with torch.autocast("cuda", dtype=HALF):
        y = gated_ffn.gated_ffn(*leaves, activation=kind)
    grads = torch.autograd.grad(y, leaves, dy)
    want = block_f64.gated_ffn(*(_np(t.detach().half()) for t in leaves), kind, _np(dy), step=1.0)
    rows = np.array([i for i in range(270) if i != 17])
    for name, g in zip(("y", *NAMES), (y, *grads)):
        off, bound = np.abs(_np(g) - want[name]), _bounds(want, name, HALF, g.dtype)
        if name == "y":
            off, bound = off[rows], bound[rows]
        assert (off <= bound).all(), (name, float((off / bound).max()))
