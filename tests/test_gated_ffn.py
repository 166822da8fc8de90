"""Gated feed-forward layer: the oracle against torch autograd in float64, the refusals, and -- on the GPU -- results and gradients against the
oracle, types and autocast, ranges of float16, graphs and streams.

Bounds.  16 bits: h, dg and du are rounded once, each by at most half a step u (bf16 2^-8, fp16 2^-11) of its value -- up to 256 tokens with a backward they are held in two parts, and
the half step is u u; up to 64 without one it is 2^-16 or less.  The roundings are independent, u / sqrt(3) of a value in the worst place of a binade (its standard deviation), so a sum of them has the
deviation u / sqrt(3) `noise` (block_f64), and 6 of these bound every element of 10^5.  In bf16 what is kept of g and u for the backward has fp16's half step, 2^-11.  Where a sum has few summands it is bounded by u of their magnitudes instead.  Beside that: the result's own half
step, and float32 sums on the tensor cores, 2^-17 of the summands' magnitudes for chains of up to 4,096 (loss_tc.cu: 1.1e-5 for positive ones).
float32: three parts are exact to 2^-24, chains of 64 summands low by under 2^-22, up to 8 chains of which are added here, and products of parts
left out: 2^-20 of the magnitudes.
"""
import numpy as np
import pytest
import torch

from oracle import block_f64

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
DTYPES = list(HALF_STEP)
NAMES = ("dx", "dw_gate", "dw_up", "dw_down")
_id = lambda d: str(d).split(".")[-1]
_np = lambda t: t.detach().double().cpu().numpy()


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
def test_oracle_matches_autograd(kind):
    g = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    x, wg, wu, wd = rand(9, 5), rand(7, 5), rand(7, 5), rand(6, 7)
    dy = torch.randn(9, 6, generator=g, dtype=torch.float64)
    f = getattr(torch.nn.functional, kind)
    y = (f(x @ wg.t()) * (x @ wu.t())) @ wd.t()
    want = torch.autograd.grad(y, (x, wg, wu, wd), dy)
    got = block_f64.gated_ffn(*(t.detach().numpy() for t in (x, wg, wu, wd)), kind, dy.numpy())
    assert np.abs(got["y"] - y.detach().numpy()).max() <= 1e-12
    for name, w in zip(NAMES, want):
        assert np.abs(got[name] - w.numpy()).max() <= 1e-12


def test_entry_points_refuse_bad_arguments_before_any_launch():
    from machinelearning_b200 import _build, _lib
    _build.build()
    lib = _lib.load()
    copies = lambda x=256, xd=2, wg=256, wu=256, wd=256, w=2, dt=2, n=10, d=64, F=128, tr=1: lib.nlfa_gated_ffn_copies(x, xd, wg, wu, wd, w, dt, n, d, F, tr)
    assert copies() == 0 and copies(x=264) == 1 and copies(wu=258) == 4 and copies(F=96) == 8 and copies(d=40) == 7
    assert copies(xd=0) == 1 and copies(w=0) == 14 and copies(xd=0, w=0, dt=0) == 15
    assert copies(xd=0, w=0, tr=0) == 0 and copies(d=40, tr=0) == 0 and copies(d=40, tr=0, n=100) == 7 and copies(d=44, tr=0) == 7
    tape = lambda n=10, d=64, F=128, o=64, dt=2, cp=0, train=1: lib.nlfa_gated_ffn_tape_bytes(n, d, F, o, dt, cp, train)
    scratch = lambda n=10, d=64, F=128, o=64, dt=2, cp=0, tr=1, b=0: lib.nlfa_gated_ffn_scratch_bytes(n, d, F, o, dt, cp, tr, b)
    assert 0 < tape(train=0) < tape() < tape(cp=15) and tape(F=0) == 0 and tape(n=-1) == 0 and tape(dt=4) == 0
    assert 0 < scratch() and 0 < scratch(b=1) and scratch(d=0) == 0

    def fwd(x=256, xd=2, wg=256, wu=256, wd=256, w=2, dt=2, act=0, n=10, d=64, F=128, o=64, y=256, cp=0, tp=256, tb=None, s=256, sb=None):
        return lib.nlfa_gated_ffn_fwd(x, xd, wg, wu, wd, w, dt, act, n, d, F, o, y, cp, 1, tp, tape() if tb is None else tb, s,
                                      scratch() if sb is None else sb, None)
    assert fwd(n=-1) == 2 and fwd(d=0) == 2 and fwd(F=0) == 2 and fwd(o=0) == 2 and fwd(d=(1 << 24) + 1) == 2 and fwd(n=(1 << 30) + 1) == 2
    assert fwd(xd=3) == 3 and fwd(w=-1) == 3 and fwd(dt=5) == 3 and fwd(act=3) == 14 and fwd(act=-1) == 14
    assert fwd(x=None) == 1 and fwd(wg=None) == 1 and fwd(wu=None) == 1 and fwd(wd=None) == 1 and fwd(y=None) == 1 and fwd(tp=None) == 1 and fwd(s=None) == 1
    assert fwd(x=257) == 6 and fwd(wd=257) == 6 and fwd(y=264) == 6 and fwd(tp=264) == 6 and fwd(s=264) == 6
    assert fwd(x=264) == 6 and fwd(d=40) == 6                    # an operand that has to be copied, and is not
    assert fwd(tb=tape() - 1) == 11 and fwd(sb=scratch() - 1) == 11
    assert fwd(n=0, x=None, y=None) == 0

    def bwd(dy=256, x=256, xd=2, wg=256, wu=256, wd=256, w=2, dt=2, act=0, n=10, d=64, F=128, o=64, cp=0, tp=256, tb=None, dx=256, dg=256, du=256,
            dd=256, s=256, sb=None):
        return lib.nlfa_gated_ffn_bwd(dy, x, xd, wg, wu, wd, w, dt, act, n, d, F, o, cp, tp, tape() if tb is None else tb, dx, dg, du, dd, s,
                                      scratch(b=1) if sb is None else sb, None)
    assert bwd(F=0) == 2 and bwd(w=9) == 3 and bwd(act=4) == 14
    assert bwd(dy=None) == 1 and bwd(x=None) == 1 and bwd(wg=None) == 1 and bwd(wu=None) == 1 and bwd(wd=None) == 1 and bwd(tp=None) == 1
    assert bwd(x=264) == 6 and bwd(wu=264) == 6 and bwd(dx=264) == 6 and bwd(dd=264) == 6 and bwd(dy=257) == 6 and bwd(s=264) == 6
    assert bwd(tb=tape() - 1) == 11 and bwd(sb=scratch(b=1) - 1) == 11
    assert bwd(dx=None, dg=None, du=None, dd=None) == 0


def test_python_call_refuses_what_it_does_not_take():
    from machinelearning_b200 import gated_ffn
    x, w = torch.randn(4, 8), torch.randn(16, 8)
    assert not gated_ffn.supports(x, w, w, w.t())
    with pytest.raises(ValueError, match="unsupported inputs"):
        gated_ffn.gated_ffn(x, w, w, w.t().contiguous())
    with pytest.raises(ValueError, match="activation"):
        gated_ffn.gated_ffn(x, w, w, w, activation="tanh")


def _inputs(dtype, n, d, F, o, seed=0, w_dtype=None, up=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed + 1000 * n + F)
    rand = lambda *s, std=1.0: torch.randn(*s, device=device, generator=g) * std
    w_dtype = w_dtype or dtype
    leaves = [rand(n, d).to(dtype), rand(F, d, std=d**-0.5).to(w_dtype), rand(F, d, std=d**-0.5).to(w_dtype), rand(o, F, std=F**-0.5).to(w_dtype)]
    return [t.requires_grad_() for t in leaves], rand(n, o, std=up)


def _bounds(want, name, dtype, out, hidden=None):
    """Elementwise, for products in `dtype` and a result of type `out`; `hidden`: half a step of h (y, dw_down) or of dg and du (the others)."""
    size = want["size_" + name]
    if dtype == torch.float32:
        return 2.0**-20 * size + HALF_STEP[out] * np.abs(want[name])
    u = HALF_STEP[dtype] if hidden is None else hidden
    if dtype == torch.bfloat16 and name in ("dx", "dw_gate", "dw_up"):       # what is kept for the backward: fp16's half step
        u = (u**2 + 2.0**-22)**0.5
    inner = np.minimum(6 / 3**0.5 * u * want["noise_" + name], 1.1 * u * size)
    return inner + 2.0**-17 * size + HALF_STEP[out] * np.abs(want[name]) + (2.0**-25 if out == torch.float16 else 0)


def _check(got, leaves, dy, kind, dtype, names=("y", *NAMES), hidden=None):
    as_seen = [_np(t.detach().to(dtype)) for t in leaves]          # (autocast rounds the operands to its type)
    want = block_f64.gated_ffn(*as_seen, kind, None if dy is None else _np(dy), step=1.0)
    for name, x in zip(names, got):
        off, bound = np.abs(_np(x).reshape(want[name].shape) - want[name]), _bounds(want, name, dtype, x.dtype, hidden)
        assert (off <= bound).all(), (name, float((off / (bound + 1e-300)).max()))


# (the last two: few tiles of long sums, whose products are formed apart; 257 rows: the first of more than one tile)
SIZES = [(1, 64, 64, 64), (1, 1, 1, 1), (2, 7, 5, 3), (64, 128, 128, 128), (65, 130, 100, 70), (129, 64, 320, 65), (256, 256, 512, 256),
         (257, 200, 129, 300), (700, 72, 1000, 64), (1000, 384, 300, 384),
         (300, 4800, 64, 72), (90, 64, 100, 5000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("n,d,F,o", SIZES)
def test_result_and_gradients(dtype, n, d, F, o):
    from machinelearning_b200 import gated_ffn
    kinds = ("silu", "gelu", "relu") if n in (65, 256) else ("silu",)
    for kind in kinds:
        leaves, dy = _inputs(dtype, n, d, F, o)
        dy = dy.to(dtype)
        y = gated_ffn.gated_ffn(*leaves, activation=kind)
        assert y.shape == (n, o) and y.dtype == dtype
        grads = torch.autograd.grad(y, leaves, dy)
        hidden = HALF_STEP[dtype]**2 if n <= 256 else None
        if kind == "relu" and dtype == torch.float32:             # (a gate's sign can hang on its sum's last bit)
            _check((y,), leaves, dy, kind, dtype, hidden=hidden)
        else:
            _check((y, *grads), leaves, dy, kind, dtype, hidden=hidden)
        again = gated_ffn.gated_ffn(*leaves, activation=kind)
        assert torch.equal(again, y) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, leaves, dy), grads))
        with torch.no_grad():
            alone = gated_ffn.gated_ffn(*leaves, activation=kind)
        _check((alone,), leaves, None, kind, dtype, hidden=2.0**-16 if n <= 64 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_id)
def test_many_tiles_and_chains(dtype):
    """More tiles than pairs of CTAs in every product, sums of more than one chain, tiles in parts; against float64 products on the GPU, in 2-norms: two
    independent roundings of u / sqrt(3) each at most, 1.2 u as a whole; float32 2^-20."""
    from machinelearning_b200 import gated_ffn
    for n, d, F, o in ((9000, 520, 1100, 4200), (5000, 4160, 700, 264)):
        leaves, dy = _inputs(dtype, n, d, F, o, seed=3)
        dy = dy.to(dtype)
        y = gated_ffn.gated_ffn(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
        wide = [t.detach().double().requires_grad_() for t in leaves]
        ref = (torch.nn.functional.silu(wide[0] @ wide[1].t()) * (wide[0] @ wide[2].t())) @ wide[3].t()
        wants = torch.autograd.grad(ref, wide, dy.double())
        most = 2.0**-20 if dtype == torch.float32 else 1.2 * HALF_STEP[dtype]
        for got, want in zip((y, *grads), (ref, *wants)):
            assert float((got.double() - want).norm() / want.norm()) <= most


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 17, 32, 33, 64, 65])
def test_a_few_tokens_without_a_backward(dtype, n):
    """The kernels of decoding steps: h is not rounded to 16 bits (its parts keep 2^-17), so the bound has no such term; and types that only autocast gives."""
    from machinelearning_b200 import gated_ffn
    for d, F, o in ((768, 2048, 768), (8, 8, 3), (64, 40, 300), (200, 1000, 17), (1032, 136, 65)):
        leaves, _ = _inputs(dtype, n, d, F, o, seed=5)
        with torch.no_grad():
            for kind in ("silu", "gelu", "relu"):
                y = gated_ffn.gated_ffn(*leaves, activation=kind)
                _check((y,), leaves, None, kind, dtype, hidden=2.0**-17 if n <= 64 else None)
                assert torch.equal(y, gated_ffn.gated_ffn(*leaves, activation=kind))
    if dtype == torch.float32:
        return
    for x_dtype in (torch.float32, torch.bfloat16, torch.float16):
        leaves, _ = _inputs(x_dtype, n, 128, 256, 64, w_dtype=torch.float32)
        with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
            y = gated_ffn.gated_ffn(*leaves)
        assert y.dtype == dtype
        _check((y,), leaves, None, "silu", dtype, hidden=2.0**-17 if n <= 64 else None)


@pytest.mark.gpu
def test_gradients_against_differences():
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.float32, 150, 96, 200, 80)
    grads = torch.autograd.grad(gated_ffn.gated_ffn(*leaves, activation="gelu"), leaves, dy)
    g = torch.Generator(device="cuda").manual_seed(5)
    for i, grad in enumerate(grads):
        v = torch.sign(grad) * (0.5 + torch.rand(grad.shape, device="cuda", generator=g)) * float(leaves[i].detach().std())
        slope, h = float((grad.double() * v.double()).sum()), 2.0**-8

        def at(sign):
            moved = [t.detach() + sign * h * v if i == j else t.detach() for j, t in enumerate(leaves)]
            return float((gated_ffn.gated_ffn(*moved, activation="gelu").double() * dy.double()).sum())
        quotient = (at(1) - at(-1)) / (2 * h)
        # along v a gate moves by up to h sqrt(d) 1.5 = 0.06; its third derivatives (below 2) enter with 0.06^2 / 6
        assert abs(quotient - slope) <= 2e-2 * abs(slope), (i, quotient, slope)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=_id)
def test_autocast(dtype):
    """float32 leaves, products and result in the autocast type, float32 gradients; a 16-bit input beside float32 weights."""
    from machinelearning_b200 import gated_ffn
    for x_dtype in (torch.float32, dtype):
        leaves, dy = _inputs(x_dtype, 300, 192, 256, 128, w_dtype=torch.float32)
        dy = dy.to(dtype)
        with torch.autocast("cuda", dtype=dtype):
            y = gated_ffn.gated_ffn(*leaves)
        assert y.dtype == dtype
        grads = torch.autograd.grad(y, leaves, dy)
        assert [g.dtype for g in grads] == [t.dtype for t in leaves]
        _check((y, *grads), leaves, dy, "silu", dtype)
    leaves, dy = _inputs(torch.bfloat16, 20, 64, 64, 64, w_dtype=torch.float32)
    with pytest.raises(ValueError, match="unsupported inputs"):
        gated_ffn.gated_ffn(*leaves)


@pytest.mark.gpu
@pytest.mark.parametrize("x_size,w_size,up", [(1.0, 1.0, 2.0**-20), (2.0**-6, 2.0**-4, 2.0**-14), (300.0, 8.0, 1.0), (30.0, 1.0, 1000.0)])
def test_float16_hidden_values_outside_the_types_range(x_size, w_size, up):
    """h up to 10^7, dg down to 10^-9: both far outside float16, whose results of such inputs are in it."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.float16, 300, 256, 384, 128, up=up)
    down = min(1.0, 1.0 / (x_size * w_size) ** 2)                  # (weights that bring y and dx back into the range)
    leaves = [(t.detach().float() * s).half().requires_grad_() for t, s in zip(leaves, (x_size, w_size, w_size, down))]
    dy = dy.half()
    y = gated_ffn.gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    ref = (torch.nn.functional.silu(wide[0] @ wide[1].t()) * (wide[0] @ wide[2].t())) @ wide[3].t()
    wants = torch.autograd.grad(ref, wide, dy.double())
    for got, want in zip((y, *grads), (ref, *wants)):
        # An element is a sum of some hundred products with h, dg or du, each of which carries an independent rounding of deviation u / sqrt(3): its error's
        # deviation is u / sqrt(3) times the root of the sum of the products' squares, which is also what the elements' own size is on
        # average (their signs are independent).  So the errors are below 1.2 u rms(want) as a whole, also of elements that are small because their products
        # cancel -- where most elements are outside float16, those that fit are such -- and 6 of these below an element's.
        want = want.detach()
        rms = 1.2 * 2.0**-11 * float(want.norm()) / want.numel()**0.5
        fits = want.abs() < 65504 - 6 * rms
        off = (got.double() - want)[fits]
        # ... and the result's own steps below its normal range
        assert float(off.norm()) <= (rms + 2.0**-25) * off.numel()**0.5 + 2.0**-12 * float(want[fits].norm())
        assert bool(torch.isinf(got[want.abs() > 65536 + 6 * rms]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["x", "w_down"])
def test_float32_values_that_round_to_the_largest_float16(where):
    """65,512 is above float16's largest value, 65,504, and is rounded to it: finite, and part of what bounds h, dg and du."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.float32, 5, 64, 64, 32)
    dy = dy.half()
    with torch.no_grad():
        if where == "x":                                           # every g and u some 512, h up to 2^20; y some 2^10
            leaves[0][:, 0] = 65512.0
            for w in leaves[1:3]:
                w[:, 0] = w[:, 0].sign() * 2.0**-7
            leaves[3] *= 2.0**-8
        else:                                                      # dg of one hidden value up to 2^18; y there is outside float16
            leaves[3][7, 11] = 65512.0
    with torch.autocast("cuda", dtype=torch.float16):
        y = gated_ffn.gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    # (what h, dg and du lose below float16's normal range is 2^-25 of 2^15 / the largest: below 2^-17 of the sums' magnitudes, which hold the largest, or
    # of one rounding's 2^-11 of the others, which are above 2^-14 of it there)
    if where == "x":
        _check((y, *grads), leaves, dy, "silu", torch.float16)
    else:
        _check(grads, leaves, dy, "silu", torch.float16, NAMES)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
def test_a_row_that_is_not_finite_stays_alone(dtype):
    """Its own y and dx, and the weights' gradients it enters; other rows' bits are what they were (in 16 bits; and in float32, where an infinity gives NaN)."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(dtype, 300, 128, 256, 64)
    dy = dy.to(dtype)
    clean = gated_ffn.gated_ffn(*leaves)
    clean_dx = torch.autograd.grad(clean, leaves[0], dy)[0]
    for bad in (float("nan"), float("inf")):
        x = leaves[0].detach().clone()
        x[17, 5] = bad
        x.requires_grad_()
        y = gated_ffn.gated_ffn(x, *leaves[1:])
        dx, dwg = torch.autograd.grad(y, (x, leaves[1]), dy)
        keep = torch.arange(300, device="cuda") != 17
        assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])
        assert not bool(torch.isfinite(y[17]).any()) and not bool(torch.isfinite(dx[17]).any()) and not bool(torch.isfinite(dwg).all())


@pytest.mark.gpu
def test_large_gates_keep_their_digits():
    """Pre-activations beyond float16 in bfloat16: they are kept for the backward with a power of two."""
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.bfloat16, 200, 128, 256, 64, up=1e-3)
    leaves = [(t.detach() * s).requires_grad_() for t, s in zip(leaves, (3e4, 40.0, 40.0, 1e-9))]
    dy = dy.bfloat16()
    y = gated_ffn.gated_ffn(*leaves)
    _check((y, *torch.autograd.grad(y, leaves, dy)), leaves, dy, "silu", torch.bfloat16)


@pytest.mark.gpu
def test_no_tokens_shapes_and_layouts():
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.bfloat16, 60, 128, 192, 64)
    want = gated_ffn.gated_ffn(*leaves)
    dy = dy.bfloat16()
    wants = torch.autograd.grad(want, leaves, dy)
    x3 = leaves[0].detach().view(3, 4, 5, 128).requires_grad_()
    y = gated_ffn.gated_ffn(x3, *leaves[1:])
    assert y.shape == (3, 4, 5, 64) and torch.equal(y.view(60, 64), want)
    (dx,) = torch.autograd.grad(y, x3, dy.view(3, 4, 5, 64))
    assert torch.equal(dx.view(60, 128), wants[0])
    # weights as a transposed view, an input with gaps, an input between 16-byte boundaries
    wide = torch.zeros(60, 200, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:131] = leaves[0].detach()
    flat = torch.zeros(60 * 128 + 8, device="cuda", dtype=torch.bfloat16)
    flat[1:60 * 128 + 1] = leaves[0].detach().reshape(-1)
    for x in (wide[:, 3:131], flat[1:60 * 128 + 1].view(60, 128)):
        args = [x.requires_grad_(), leaves[1].detach().t().contiguous().t().requires_grad_(), *leaves[2:]]
        y = gated_ffn.gated_ffn(*args)
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, args, dy), wants))
    # a gradient that is expanded, and one of another type
    y = gated_ffn.gated_ffn(*leaves)
    got = torch.autograd.grad(y.float().sum(), leaves)
    same = torch.autograd.grad(gated_ffn.gated_ffn(*leaves), leaves, torch.ones_like(dy))
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    empty = leaves[0].detach()[:0].requires_grad_()
    y = gated_ffn.gated_ffn(empty, *leaves[1:])
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, (empty, *leaves[1:]), dy[:0])
    assert grads[0].shape == (0, 128) and all(bool((g == 0).all()) for g in grads)
    vector = leaves[0].detach()[3]
    assert torch.equal(gated_ffn.gated_ffn(vector, *leaves[1:])[None], gated_ffn.gated_ffn(vector[None], *leaves[1:]))


@pytest.mark.gpu
def test_gradients_that_are_not_wanted():
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.bfloat16, 400, 128, 256, 192)
    dy = dy.bfloat16()
    want = torch.autograd.grad(gated_ffn.gated_ffn(*leaves), leaves, dy)
    for mask in range(1, 15):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(leaves)]
        asked = [i for i in range(4) if mask >> i & 1]
        got = torch.autograd.grad(gated_ffn.gated_ffn(*some), [some[i] for i in asked], dy)
        for i, g in zip(asked, got):
            # (a tile may be formed in another number of parts: float32 sums in another order)
            assert float((g.float() - want[i].float()).norm() / want[i].float().norm()) <= 2.0**-9


@pytest.mark.gpu
def test_graph_capture_and_side_stream():
    from machinelearning_b200 import gated_ffn
    for dtype in (torch.bfloat16, torch.float16):
        leaves, dy = _inputs(dtype, 500, 128, 320, 128)
        dy = dy.to(dtype)

        def step():
            y = gated_ffn.gated_ffn(*leaves)
            return y.detach(), *torch.autograd.grad(y, leaves, dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            on_side = step()
        torch.cuda.current_stream().wait_stream(side)
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(on_side, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for factor in (1.0, 0.25):                                # replayed on other values, beside an eager call
            with torch.no_grad():
                leaves[0].mul_(factor)
            graph.replay()
            eager = step()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("auto", [False, True])
def test_compiled_caller_keeps_one_graph(auto):
    from machinelearning_b200 import flash_cuda, gated_ffn
    assert flash_cuda.is_available()
    leaves, dy = _inputs(torch.float32 if auto else torch.bfloat16, 70, 64, 128, 64)
    dy = dy.bfloat16()

    def call(x, a, b, c):
        return gated_ffn.gated_ffn(x, a, b, c) * 2

    def run(f):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=auto):
            y = f(*leaves)
        return y, *torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(run(torch.compile(call, fullgraph=True)), run(call)))


@pytest.mark.gpu
def test_saved_tensors_that_change_raise_and_moved_ones_do_not():
    from machinelearning_b200 import gated_ffn
    leaves, dy = _inputs(torch.bfloat16, 50, 64, 128, 64)
    dy = dy.bfloat16()
    x = leaves[0] * 1
    y = gated_ffn.gated_ffn(x, *leaves[1:])
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)
    want = torch.autograd.grad(gated_ffn.gated_ffn(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = gated_ffn.gated_ffn(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
    up = dy.detach().requires_grad_()
    (dx,) = torch.autograd.grad(gated_ffn.gated_ffn(*leaves), leaves[0], up, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
def test_refusals_on_the_device():
    from machinelearning_b200 import gated_ffn
    (x, wg, wu, wd), _ = _inputs(torch.bfloat16, 4, 64, 96, 32)
    for bad in ((x[:, :32], wg, wu, wd), (x, wg, wu[:90], wd), (x, wg, wu, wd[:, :90]), (x, wg, wu.half(), wd), (x.cpu(), wg, wu, wd),
                (x, wg.cpu(), wu, wd), (x.double(), wg.double(), wu.double(), wd.double()), (x, wg[0], wu[0], wd)):
        with pytest.raises(ValueError, match="unsupported inputs"):
            gated_ffn.gated_ffn(*bad)
