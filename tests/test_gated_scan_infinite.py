"""Gated recurrence: what is not finite stays in the states, and in the gradients, up to the next reset -- however large the gates are that it goes
through, and however the sequence is cut into runs and segments.

The factors of many steps' states underflow (gates of 20 within some 5 steps of float32's range, ordinary ones within some 150): zero times infinity is
NaN, so nothing that is not finite may come out finite; only a reset leaves it out.  Channels have nothing to do with one another: the others keep their bits.
"""
import numpy as np
import pytest
import torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
_id = lambda d: str(d).split(".")[-1]
# one run; runs of one CTA; runs of several stretches; segments, of pairs and of single channels
PLANS = [(2, 7, 64), (2, 40, 8), (3, 300, 72), (1, 4100, 64), (1, 2100, 33)]
# segments so long that the factors of ordinary gates underflow within one
LONG = (1, 16384, 1024)
BAD = [float("nan"), float("inf"), -float("inf")]


def _inputs(B, T, D, dtype, gates):
    g = torch.Generator(device="cuda").manual_seed(T + D)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return [(rand(B, T, D) + gates).to(dtype), rand(B, T, D).to(dtype), rand(B, D), rand(B, T, D).to(dtype), rand(B, D)]


def _run(gate, value, state, dh, dlast, **kw):
    from machinelearning_b200 import gated_scan
    leaves = [t.detach().clone().requires_grad_() for t in (gate, value, state)]
    h, last = gated_scan.gated_scan(*leaves, **kw)
    return h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (dh, dlast))


def _no(t):
    return not bool(torch.isfinite(t).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("gates", [20.0, 0.0])
@pytest.mark.parametrize("B,T,D", [*PLANS, LONG])
def test_what_is_not_finite_stays(dtype, gates, B, T, D):
    for reset_at in (None, 2 * T // 3):
        gate, value, state, dh, dlast = _inputs(B, T, D, dtype, gates)
        reset = torch.zeros(B, T, dtype=torch.bool, device="cuda")
        if reset_at is not None:
            reset[:, reset_at] = True
        kw = {"reset": reset if reset_at is not None else None}
        end = T if reset_at is None else reset_at
        begin = 0 if reset_at is None else reset_at
        clean = _run(gate, value, state, dh, dlast, **kw)
        c, others = 3, torch.arange(D, device="cuda") != 3
        for bad in BAD:
            # a state, or one value, that is not finite: the states behind it, up to the reset
            for at in (-1, 1, T // 2):
                v, s = value.clone(), state.clone()
                (s if at < 0 else v[:, at])[:, c] = bad
                h, last, *_ = _run(gate, v, s, dh, dlast, **kw)
                assert _no(h[:, max(at, 0):end, c])
                if reset_at is None:
                    assert _no(last[:, c])
                else:
                    assert torch.equal(h[:, end:], clean[0][:, end:]) and torch.equal(last, clean[1])
                assert torch.equal(h[..., others], clean[0][..., others]) and torch.equal(last[:, others], clean[1][:, others])
            # a gradient that is not finite: those of the steps in front of it, down to the reset
            for at in (T, T - 2, T - T // 6):
                d, l = dh.clone(), dlast.clone()
                (l if at == T else d[:, at])[:, c] = bad
                _, _, dz, dv, ds = _run(gate, value, state, d, l, **kw)
                assert _no(dv[:, begin:min(at + 1, T), c])
                if reset_at is None:
                    assert _no(ds[:, c])
                else:
                    assert torch.equal(dv[:, :begin], clean[3][:, :begin]) and torch.equal(dz[:, :begin], clean[2][:, :begin]) and torch.equal(ds, clean[4])
                assert all(torch.equal(a[..., others], b[..., others]) for a, b in zip((dz, dv, ds), clean[2:]))


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,D", PLANS)
def test_padding_leaves_a_state_that_is_not_finite_as_it_is(B, T, D):
    gate, value, state, dh, dlast = _inputs(B, T, D, torch.bfloat16, 0.0)
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    state[:, 0], state[:, 1] = float("inf"), -float("inf")
    h, last, _, _, ds = _run(gate, value, state, dh, dlast, lengths=lengths)
    assert torch.equal(last, state) and torch.equal(ds, dlast) and not bool(h.any())
    state[:, 2] = float("nan")
    assert bool(torch.isnan(_run(gate, value, state, dh, dlast, lengths=lengths)[1][:, 2]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("B,T,D", PLANS)
def test_finite_states_behind_products_that_underflow(dtype, B, T, D):
    """Gates of 15 to 25 and the oracle: nothing of a state is left a few steps on.  Bounds as for states of a short memory (test_gated_scan.py)."""
    from oracle import block_f64
    from test_gated_scan import _check
    gate, value, state, dh, dlast = _inputs(B, T, D, dtype, 20.0)
    np_ = lambda t: t.double().cpu().numpy()
    reset = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    reset[:, T // 2] = True
    for r in (None, reset):
        want = block_f64.gated_scan(np_(gate), np_(value), np_(state), "none", None if r is None else r.cpu().numpy(), None, np_(dh), np_(dlast))
        _check(_run(gate, value, state, dh, dlast, reset=r), want, dtype, T)


@pytest.mark.gpu
def test_the_mixer_gives_what_tensor_operations_give():
    """whole_model's mixer in tensor operations and through the kernel: infinities in the same places, and equal states where gates' products underflow."""
    from machinelearning_b200 import gated_scan, whole_model
    gate, value, state, _, _ = _inputs(2, 700, 64, torch.float32, 25.0)
    for at in (None, 100):
        v = value.clone()
        if at is not None:
            v[0, at, 5] = float("inf")
        plain, plain_last = whole_model.plain_scan(gate, v, state)
        h, last = gated_scan.gated_scan(gate, v, state, activation="positive")
        finite = torch.isfinite(plain)
        assert torch.equal(torch.isfinite(h), finite) and torch.equal(torch.isfinite(last), torch.isfinite(plain_last))
        # both: 1 - s below 2^-32, so h is f up to two roundings of its size
        assert bool(((h - plain).abs()[finite] <= 2.0**-21 * (plain.abs()[finite] + 1)).all())
        assert np.isfinite(float(h[finite].sum()))
