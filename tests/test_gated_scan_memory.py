"""Gated recurrence: states that last for a million steps keep their digits, and so do the gradients that go back as far.

Constant gates, so that every result has a closed form: s = sigmoid(gate) in float64, and (1 - s)^t.  1 - s itself, in float32, is rounded by up to 2^-25, always
in the same direction: states multiplied with it, step by step or run by run, would be off by up to 2^-25 T, 3% in 2^20 steps (2.4% at a gate of -14.125).

Bounds, with u = 2^-24.  s has a relative error of 2^-21 (float32) or 2^-19 (16 bits, |gate| < 16), as in test_gated_scan.py: t s of that in
(1 - s)^t.  What is left out of a state over a run of up to 16 steps is a sum of products each rounded twice, 2^-19 of it, and joined over up to 60 runs of a segment with three
roundings each, 2^-17: t s 2^-17 at most.  Where a run, or a segment, is entered the state is rounded once, by u: N u for N of them in front, and u for each of the up to 16 steps of its own run.
Results of 16 bits: half a step.
"""
import numpy as np
import pytest
import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
GATES = [-14.125, -13.875, -13.8125, -12.3125, -11.0, -9.0, -6.5, -2.0]      # (all exact in bfloat16)
# B, T, D, and how many runs and segments a state is rounded at
PLANS = [(1, 1 << 20, 8, 1400), (1, 1 << 18, 7, 1400), (80, 1 << 15, 64, None), (100, 1 << 15, 64, None)]
_id = lambda d: str(d).split(".")[-1]
_np = lambda t: t.detach().double().cpu().numpy()


def _s(D):
    return 1 / (1 + np.exp(-np.array([GATES[i % 8] for i in range(D)])))


def _near(got, want, part):
    """`part`: of want, with half a step of got's type; what is below float32's normal range (float16's: its own) is not looked at."""
    low = 2.0**-24 if got.dtype == torch.float16 else 2.0**-120
    off = np.abs(_np(got) - want)
    bound = np.abs(want) * (np.expm1(np.minimum(part, 600.0)) + HALF_STEP[got.dtype]) + low
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF_STEP), ids=_id)
@pytest.mark.parametrize("B,T,D,entered", PLANS)
def test_states_and_gradients_of_slow_gates(dtype, B, T, D, entered):
    from machinelearning_b200 import gated_scan
    run = 8 if dtype == torch.float32 else 16
    s = _s(D)
    row = torch.tensor([GATES[i % 8] for i in range(D)], device="cuda", dtype=dtype)
    gate, zero, one = (t.expand(B, T, D) for t in (row, torch.zeros_like(row), torch.ones_like(row)))
    entered = (T // run if entered is None else entered) + 17
    t = np.array([1, 2, T // 3, T - 1, T])[:, None]
    off = t * s * ((2.0**-21 if dtype == torch.float32 else 2.0**-19) + 2.0**-17) / (1 - s) + entered * 2.0**-24
    left = np.exp(t * np.log1p(-s))                                # of a state, t steps on
    at = torch.tensor(t[:, 0] - 1, device="cuda")

    # a state of one and no values: what is left of it
    state = torch.ones(B, D, device="cuda", requires_grad=True)
    h, last = gated_scan.gated_scan(gate, zero, state)
    _near(h[:, at], np.broadcast_to(left, (B, 5, D)), off)
    _near(last, np.broadcast_to(left[-1], (B, D)), off[-1])
    (ds,) = torch.autograd.grad(last, state, torch.ones_like(last))
    _near(ds, np.broadcast_to(left[-1], (B, D)), off[-1])
    del h, last
    # values of one and no state: the rest (its error is that of s and of what is entered, in proportion)
    grown = -np.expm1(t * np.log1p(-s))
    h, last = gated_scan.gated_scan(gate, one)
    part = (2.0**-21 if dtype == torch.float32 else 2.0**-19) + 2.0**-17 + entered * 2.0**-24
    _near(h[:, at], np.broadcast_to(grown, (B, 5, D)), part)
    _near(last, np.broadcast_to(grown[-1], (B, D)), part)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 7])
def test_gradients_of_gates_and_values_along_a_slow_sequence(D):
    """float32, one sequence in segments: dv_t = (1 - s)^(T - t) s of the last state, dz_t = -(1 - s)^T s for a state of one."""
    from machinelearning_b200 import gated_scan
    T = 1 << 20
    s = _s(D)
    row = torch.tensor([GATES[i % 8] for i in range(D)], device="cuda")
    gate, value = row.expand(1, T, D).contiguous().requires_grad_(), torch.zeros(1, T, D, device="cuda", requires_grad=True)
    state = torch.ones(1, D, device="cuda")
    _, last = gated_scan.gated_scan(gate, value, state)
    dz, dv = torch.autograd.grad(last, (gate, value), torch.ones_like(last))
    t = np.array([1, 5, T // 2, T - 7, T])[:, None]
    at = torch.tensor(t[:, 0] - 1, device="cuda")
    # G from behind and h from in front are both as the states above; s itself, 1 - s, and three products
    off = T * s * (2.0**-21 + 2.0**-17) / (1 - s) + 2 * 1417 * 2.0**-24 + 2.0**-20
    _near(dv[0, at], np.exp((T - t) * np.log1p(-s)) * s, off)
    _near(dz[0, at], -np.exp(T * np.log1p(-s)) * s * np.ones_like(t), off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF_STEP), ids=_id)
def test_slow_and_fast_gates_side_by_side(dtype):
    """Gates that go from slow to fast along the sequence, so that runs and segments keep from all of a state to nothing of it; resets on the way."""
    from machinelearning_b200 import gated_scan
    B, T, D = 1, 6000, 24
    g = torch.Generator(device="cuda").manual_seed(8)
    gate = (torch.linspace(-13, 6, T, device="cuda")[:, None] + 3 * torch.rand(D, device="cuda", generator=g)).to(dtype)[None]
    reset = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    reset[:, [700, 701, 3000]] = True
    z = _np(gate)[0]
    keep = np.log1p(-1 / (1 + np.exp(-z)))
    run, logs = np.zeros(D), np.zeros((T, D))
    for t in range(T):
        run = run + keep[t]
        logs[t] = run
    slow = np.exp(z)                                               # >= s: what its error is taken of
    off = np.cumsum(slow, 0) * (2.0**-18 + 2.0**-17) + 1417 * 2.0**-24
    for r in (None, reset):
        want = np.exp(logs) if r is None else np.where(np.arange(T)[:, None] < 700, np.exp(logs), 0.0)
        h, last = gated_scan.gated_scan(gate, torch.zeros_like(gate), torch.ones(B, D, device="cuda"), reset=r)
        _near(h[0], want, off)
        _near(last[0], want[-1], off[-1])
