"""Gated feed-forward layer, a few tokens of wide layers without a backward: long sums of one sign are not low by what the tensor core cuts off.

The tensor core adds by truncation, so a chain of positive summands comes out low, by some 8.6e-10 a summand in float32's place (4,096 of them: 1.1e-5).  Chains are cut and their sums added in
float32, rounded: float32 chains of 64 summands and less are low by 2^-24; g, u and the sum over hidden values have three such shares, below 2^-22 together.  Roundings of additions are independent: over up
to 128 of growing sums 2^-24 / sqrt(3) sqrt(128 / 3) is their deviation, 6 of these 2^-20.5; in g and u (over 512 of them 2^-19.5) they cancel over the hidden values, 64 and more.  The parts of a
value are exact to 2^-24.  Together below 2^-20 of y, where F / 16 has 64 chains and less.  16 bits: chains of 2,048 summands and less, below 2^-18 three times, beside the result's half step: below 2^-16 of y.
"""
import numpy as np
import pytest
import torch

from oracle import block_f64
from test_gated_ffn import DTYPES, HALF_STEP, _id, _np


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("n,d,F,o", [(1, 4096, 8192, 40), (16, 4096, 4096, 24), (3, 16384, 256, 16), (16, 64, 32768, 16), (9, 65536, 64, 8), (64, 16384, 128, 16)])
def test_long_sums_of_one_sign(dtype, n, d, F, o):
    from machinelearning_b200 import gated_ffn
    g = torch.Generator(device="cuda").manual_seed(n + d)
    some = lambda *s, size: ((0.5 + torch.rand(*s, device="cuda", generator=g)) * size).to(dtype)
    x, wg, wu, wd = some(n, d, size=1.0), some(F, d, size=1 / d), some(F, d, size=1 / d), some(o, F, size=1 / F)
    if dtype == torch.float16:                                     # (weights of 1 / d would be below its normal range)
        x, wg, wu, wd = some(n, d, size=1.0), some(F, d, size=2.0**-10), some(F, d, size=2.0**-10), some(o, F, size=2.0**-12)
    with torch.no_grad():
        y = gated_ffn.gated_ffn(x, wg, wu, wd, activation="relu")
    want = block_f64.gated_ffn(*(_np(t) for t in (x, wg, wu, wd)), "relu")["y"]
    assert want.min() > 0 and want.max() < 6e4
    off = np.abs(_np(y) - want)
    most = HALF_STEP[dtype] + (2.0**-20 if dtype == torch.float32 else 2.0**-16)
    assert (off <= most * want).all(), float((off / want).max() / most)
