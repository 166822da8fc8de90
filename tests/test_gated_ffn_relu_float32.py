"""Gated feed-forward layer in float32 with relu: all gradients against the oracle.

Relu's slope jumps at zero, so no gate may be so near it that its sign hangs on the rounding of a sum: tokens with a gate within twice the sum's bound, 2^-20 of its summands'
magnitudes, are drawn anew.
"""
import pytest
import torch

from test_gated_ffn import NAMES, _check, _inputs


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,F,o", [(2, 7, 5, 3), (65, 130, 100, 70), (256, 256, 512, 256), (257, 200, 129, 300), (700, 72, 1000, 64), (300, 2400, 64, 72)])
def test_gradients(n, d, F, o):
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.float32, n, d, F, o, seed=11)
    g = torch.Generator(device="cuda").manual_seed(n)
    with torch.no_grad():
        x, wg = leaves[0], leaves[1].double()
        for _ in range(100):
            near = ((x.double() @ wg.t()).abs() <= 2.0**-19 * (x.double().abs() @ wg.abs().t())).any(1)
            if not bool(near.any()):
                break
            x[near] = torch.randn(int(near.sum()), d, device="cuda", generator=g)
        else:
            raise AssertionError("gates at zero")
    y = gated_ffn.gated_ffn(*leaves, activation="relu")
    _check((y, *torch.autograd.grad(y, leaves, dy)), leaves, dy, "relu", torch.float32, ("y", *NAMES))
