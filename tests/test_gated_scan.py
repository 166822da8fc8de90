"""Gated recurrence: the oracle against torch autograd in float64, the refusals, and -- on the GPU -- states and gradients against the
oracle, resets and padding that hide what they cover, decoding, graphs and streams.

Bounds.  s and 1 - s: the smaller is e / (1 + e); e comes with 2^-22 of the hardware's exponential (16-bit inputs) and the rounding of its argument, |z| 1.44
times 2^-24 (|z| < 16: 2^-20), two more roundings: u_s = 2^-19 of it; float32 inputs: expf's two units (2^-22), sum and quotient: 2^-21.  An error of
u_s in one gate moves h by u_s s (f - h); over the steps that a state lasts these shares s add up to at most about 1 + the ones that
are large: 4 u_s of the magnitudes.  A step's own rounding, 2^-24 of h twice, is forgotten after 1 / s steps: at most 2^-23 (memory) of the
magnitudes, memory = min(T, max 1 / s).  Runs joined through their maps round as many times.  A gradient has the recurrence twice (of h and of G).
16-bit outputs: half a step.
"""
import numpy as np
import pytest
import torch

from oracle import block_f64

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
DTYPES = list(HALF_STEP)
_id = lambda d: str(d).split(".")[-1]


def _torch_scan(gate, value, state, activation, reset, lengths):
    """The definition, step by step on tensors."""
    B, T, D = gate.shape
    h = gate.new_zeros(B, D) if state is None else state
    f = value if activation == "none" else torch.where(value < 0, torch.sigmoid(value), value + 0.5)
    s, out = torch.sigmoid(gate), []
    for t in range(T):
        before = h if reset is None else torch.where(reset[:, t, None], torch.zeros_like(h), h)
        new = (1 - s[:, t]) * before + s[:, t] * f[:, t]
        live = torch.ones(B, 1, dtype=torch.bool) if lengths is None else (lengths > t)[:, None]
        out.append(torch.where(live, new, torch.zeros_like(new)))
        h = torch.where(live, new, h)
    return (torch.stack(out, 1) if T else gate.new_zeros(B, 0, D)), h


@pytest.mark.parametrize("activation", ["none", "positive"])
def test_oracle_matches_autograd(activation):
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    gate, value, state = (t.requires_grad_() for t in (rand(3, 9, 4), rand(3, 9, 4), rand(3, 4)))
    reset = torch.rand(3, 9, generator=g) < 0.2
    lengths = torch.tensor([9, 0, 5])
    dh, dlast = rand(3, 9, 4), rand(3, 4)
    h, last = _torch_scan(gate, value, state, activation, reset, lengths)
    want = torch.autograd.grad((h, last), (gate, value, state), (dh, dlast))
    got = block_f64.gated_scan(gate.detach(), value.detach(), state.detach(), activation, reset, lengths, dh, dlast)
    for a, b in zip((got["h"], got["last"], got["dgate"], got["dvalue"], got["dstate"]), (h.detach(), last.detach(), *want)):
        assert np.abs(a - b.numpy()).max() <= 1e-13


def test_entry_points_refuse_bad_arguments_before_any_launch():
    from machinelearning_b200 import _build, _lib
    _build.build()
    lib = _lib.load()

    def fwd(z=256, v=256, dt=2, state=None, reset=None, lengths=None, lb=0, act=0, B=2, T=40, D=8, h=256, last=256, tape=256, tb=None,
            s=256, sb=1 << 20):
        need = lib.nlfa_gated_scan_tape_bytes(2, 40, 8, 2)
        return lib.nlfa_gated_scan_fwd(z, T * D, D, v, T * D, D, dt, state, reset, lengths, lb, act, B, T, D, h, last, tape, need if tb is None else tb,
                                       s, sb, None)
    assert lib.nlfa_gated_scan_tape_bytes(2, 40, 8, 2) == 2 * 3 * 8 * 4 and lib.nlfa_gated_scan_tape_bytes(2, 40, 8, 0) == 2 * 5 * 8 * 4
    assert lib.nlfa_gated_scan_tape_bytes(2, -1, 8, 2) == 0 and lib.nlfa_gated_scan_scratch_bytes(2, 40, 8, 9) == 0
    assert fwd(B=-1) == 2 and fwd(T=-1) == 2 and fwd(D=-1) == 2 and fwd(T=(1 << 30) + 1) == 2
    assert fwd(dt=3) == 3 and fwd(act=2) == 14 and fwd(lengths=256, lb=2) == 14
    assert fwd(z=None) == 1 and fwd(v=None) == 1 and fwd(h=None) == 1 and fwd(last=None) == 1
    assert fwd(z=257) == 6 and fwd(v=257) == 6 and fwd(h=258, dt=0) == 6 and fwd(state=258) == 6 and fwd(last=258) == 6 and fwd(lengths=260, lb=8) == 6
    assert fwd(tb=191) == 11 and fwd(s=264) == 6
    assert fwd(B=0, z=None, v=None, h=None, last=None) == 0 and fwd(D=0) == 0

    def bwd(z=256, v=256, dt=2, dh=256, dlast=256, lengths=None, lb=0, act=0, B=2, T=40, D=8, tape=256, tb=192, dz=256, dv=256, ds=256,
            s=256, sb=1 << 20):
        return lib.nlfa_gated_scan_bwd(dh, dlast, z, T * D, D, v, T * D, D, dt, None, lengths, lb, act, B, T, D, tape, tb, dz, dv, ds, s, sb, None)
    assert bwd(B=-1) == 2 and bwd(dt=7) == 3 and bwd(act=-1) == 14 and bwd(lengths=256, lb=3) == 14
    assert bwd(z=None) == 1 and bwd(v=None) == 1 and bwd(tape=None) == 1
    assert bwd(dh=257) == 6 and bwd(dz=257) == 6 and bwd(dv=257) == 6 and bwd(dlast=258) == 6 and bwd(ds=258) == 6 and bwd(tape=258) == 6
    assert bwd(tb=191) == 11 and bwd(dz=None, dv=None, ds=None) == 0 and bwd(B=0) == 0


def test_python_call_refuses_what_it_does_not_take():
    from machinelearning_b200 import gated_scan
    z = torch.randn(2, 5, 8)
    assert not gated_scan.supports(z, z)
    with pytest.raises(ValueError, match="unsupported inputs"):
        gated_scan.gated_scan(z, z)
    with pytest.raises(ValueError, match="activation"):
        gated_scan.gated_scan(z, z, activation="tanh")


def _inputs(B, T, D, dtype, seed=0, joint=False, bias=(-4.0, 1.0)):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * T + D)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    lo, hi = bias
    gate = rand(B, T, D) + lo + (hi - lo) * torch.rand(D, device="cuda", generator=g)
    value = rand(B, T, D)
    if joint:
        both = torch.cat((gate, value), 2).to(dtype)
        gate, value = both[..., :D], both[..., D:]
    else:
        gate, value = gate.to(dtype), value.to(dtype)
    reset = torch.rand(B, T, device="cuda", generator=g) < 3.0 / (T + 3)
    lengths = torch.randint(0, T + 1, (B,), device="cuda", generator=g)
    return gate, value, rand(B, D), reset, lengths, rand(B, T, D).to(dtype), rand(B, D)


def _check(got, want, dtype, T, what=("h", "last", "dgate", "dvalue", "dstate")):
    memory = min(T, want["memory"])
    u = 4 * (2.0**-21 if dtype == torch.float32 else 2.0**-19) + 2.0**-23 * memory
    for name, x in zip(what, got):
        if x is None:
            continue
        # the gradient of a gate has errors of G, h and of s (1 - s); that of a value errors of G and s
        parts = {"h": 1, "last": 1, "dgate": 3, "dvalue": 2, "dstate": 1}[name]
        bound = HALF_STEP[x.dtype] * np.abs(want[name]) + parts * u * want["size_" + name] + (2.0**-25 if x.dtype == torch.float16 else 0)
        off = np.abs(x.detach().double().cpu().numpy() - want[name])
        assert (off <= bound * 1.0001).all(), (name, float((off / (bound + 1e-300)).max()))


SIZES = [(1, 1, 1), (2, 1, 64), (5, 2, 7), (3, 15, 33), (2, 16, 64), (1, 17, 2), (2, 63, 66), (2, 64, 65), (1, 65, 130), (2, 129, 30), (2, 513, 34),
         (1, 1100, 70), (1, 2500, 3), (1, 1300, 136), (40, 70, 520)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("B,T,D", SIZES)
def test_states_and_gradients(dtype, B, T, D):
    from machinelearning_b200 import gated_scan
    for activation, masks, joint, with_state in (("none", "", False, True), ("positive", "reset lengths", True, True), ("none", "reset", True, False),
                                                 ("positive", "lengths", False, True)):
        gate, value, state, reset, lengths, dh, dlast = _inputs(B, T, D, dtype, joint=joint)
        leaves = [t.detach().requires_grad_() for t in (gate, value, state)]
        if not with_state:
            leaves[2] = None
        kw = {"reset": reset if "reset" in masks else None, "lengths": lengths if "lengths" in masks else None}
        h, last = gated_scan.gated_scan(*leaves, activation=activation, **kw)
        assert h.dtype == dtype and last.dtype == torch.float32 and h.shape == gate.shape and last.shape == (B, D)
        grads = torch.autograd.grad((h, last), [t for t in leaves if t is not None], (dh, dlast))
        cpu = lambda t: None if t is None else t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()
        want = block_f64.gated_scan(cpu(gate), cpu(value), cpu(leaves[2]), activation, *(cpu(t) for t in kw.values()), cpu(dh), cpu(dlast))
        _check((h, last, *grads, *([None] if not with_state else [])), want, dtype, T)
        assert (lambda a, b: torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]))(
            gated_scan.gated_scan(*leaves, activation=activation, **kw), (h, last))
        with torch.no_grad():                                     # without a tape: the same
            again = gated_scan.gated_scan(*leaves, activation=activation, **kw)
        assert torch.equal(again[0], h) and torch.equal(again[1], last)


@pytest.mark.gpu
@pytest.mark.parametrize("only", ["h", "last"])
def test_gradients_of_one_output(only):
    from machinelearning_b200 import gated_scan
    gate, value, state, reset, _, dh, dlast = _inputs(2, 200, 36, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (gate, value, state)]
    h, last = gated_scan.gated_scan(*leaves, reset=reset)
    grads = torch.autograd.grad(h if only == "h" else last, leaves, dh if only == "h" else dlast)
    np_ = lambda t: t.detach().double().cpu().numpy()
    want = block_f64.gated_scan(np_(gate), np_(value), np_(state), "none", reset.cpu().numpy(), None, np_(dh) if only == "h" else None,
                                np_(dlast) if only == "last" else None)
    _check((None, None, *grads), want, torch.float32, 200)


@pytest.mark.gpu
def test_gradients_that_are_not_wanted():
    from machinelearning_b200 import gated_scan
    gate, value, state, reset, lengths, dh, dlast = _inputs(2, 90, 40, torch.bfloat16)
    every = [t.detach().requires_grad_() for t in (gate, value, state)]
    want = torch.autograd.grad(gated_scan.gated_scan(*every, reset=reset, lengths=lengths), every, (dh, dlast))
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((gate, value, state))]
        (got,) = torch.autograd.grad(gated_scan.gated_scan(*leaves, reset=reset, lengths=lengths), leaves[i], (dh, dlast))
        assert torch.equal(got, want[i])


@pytest.mark.gpu
def test_gradients_against_differences():
    """The directional derivative of a sum of h and last against its difference quotient, float32."""
    from machinelearning_b200 import gated_scan
    gate, value, state, reset, lengths, dh, dlast = _inputs(2, 150, 20, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (gate, value, state)]
    kw = {"activation": "positive", "reset": reset, "lengths": lengths}
    grads = torch.autograd.grad(gated_scan.gated_scan(*leaves, **kw), leaves, (dh, dlast))
    g = torch.Generator(device="cuda").manual_seed(3)
    for i, grad in enumerate(grads):
        v = torch.sign(grad) * (0.5 + torch.rand(grad.shape, device="cuda", generator=g))
        if i == 1:                                                # steps that do not cross the bend of f at zero
            v = torch.where(value.abs() < 2.0**-5, torch.zeros_like(v), v)
        slope = float((grad.double() * v.double()).sum())

        def at(sign):
            moved = [t.detach() + sign * 2.0**-7 * v if i == j else t.detach() for j, t in enumerate(leaves)]
            h, last = gated_scan.gated_scan(*moved, **kw)
            return float((h.double() * dh.double()).sum() + (last.double() * dlast.double()).sum())
        quotient = (at(1) - at(-1)) * 2.0**6
        # third derivatives of sigmoids are below 1/8 and enter with (1.5 / 128)^2 / 6; h's own 2^-17 over the step
        assert abs(quotient - slope) <= 2e-2 * abs(slope), (i, quotient, slope)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40, 600])
def test_a_reset_hides_what_was_before_and_padding_hides_what_it_holds(T):
    from machinelearning_b200 import gated_scan
    gate, value, state, _, _, dh, dlast = _inputs(3, T + 30, 48, torch.bfloat16)
    reset = torch.zeros(3, T + 30, dtype=torch.bool, device="cuda")
    reset[:, T] = True
    lengths = torch.tensor([T + 30, T + 11, T + 1], device="cuda")

    def run(bad):
        z, v, s, d = gate.clone(), value.clone(), state.clone(), dh.clone()
        if bad is not None:
            s[:] = bad
            v[:, :T] = bad                                        # states before the reset are not finite
            for b, n in enumerate(lengths.tolist()):
                z[b, n:], v[b, n:], d[b, n:] = bad, bad, bad
        leaves = [t.requires_grad_() for t in (z, v, s)]
        h, last = gated_scan.gated_scan(*leaves, reset=reset, lengths=lengths)
        return h, last, *torch.autograd.grad((h, last), leaves, (d, dlast))
    clean = run(None)
    for bad in (float("nan"), float("inf"), -float("inf")):
        got = run(bad)
        assert torch.equal(got[0][:, T:], clean[0][:, T:]) and torch.equal(got[1], clean[1])
        assert torch.equal(got[2][:, T:], clean[2][:, T:]) and torch.equal(got[3][:, T:], clean[3][:, T:])
    for b, n in enumerate(lengths.tolist()):
        assert all(bool((clean[i][b, n:] == 0).all()) for i in (0, 2, 3))


@pytest.mark.gpu
def test_lengths_outside_the_sequence_and_no_steps():
    from machinelearning_b200 import gated_scan
    gate, value, state, _, _, dh, dlast = _inputs(4, 33, 10, torch.float32)
    whole = gated_scan.gated_scan(gate, value, state)
    for kind in (torch.int32, torch.int64):
        lengths = torch.tensor([33, 4000, 0, -5], device="cuda", dtype=kind)
        h, last = gated_scan.gated_scan(gate, value, state, lengths=lengths)
        assert torch.equal(h[:2], whole[0][:2]) and torch.equal(last[:2], whole[1][:2])
        assert bool((h[2:] == 0).all()) and torch.equal(last[2:], state[2:])
    none = [t[:, :0].detach().requires_grad_() for t in (gate, value)]
    s = state.detach().requires_grad_()
    h, last = gated_scan.gated_scan(*none, s)
    dz, dv, ds = torch.autograd.grad((h, last), (*none, s), (dh[:, :0], dlast))
    assert h.shape == (4, 0, 10) and torch.equal(last, s) and torch.equal(ds, dlast) and dz.shape == dv.shape == (4, 0, 10)
    h, last = gated_scan.gated_scan(gate[:0], value[:0])
    assert h.shape == (0, 33, 10) and last.shape == (0, 10)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
def test_step_by_step_is_the_whole(dtype):
    """Chunks of any lengths, single tokens among them, each from the state that the one before left."""
    from machinelearning_b200 import gated_scan
    gate, value, state, reset, _, _, _ = _inputs(3, 150, 72, dtype)
    np_ = lambda t: t.double().cpu().numpy()
    want = block_f64.gated_scan(np_(gate), np_(value), np_(state), "positive", reset.cpu().numpy())
    s, t, out = state, 0, []
    for n in (1, 1, 70, 1, 16, 17, 1, 43):
        h, s = gated_scan.gated_scan(gate[:, t:t + n], value[:, t:t + n], s, activation="positive", reset=reset[:, t:t + n])
        out.append(h)
        t += n
    assert t == 150
    _check((torch.cat(out, 1), s), want, dtype, 150)


@pytest.mark.gpu
def test_a_long_memory_keeps_its_digits():
    """Gates of 1e-6 over 20,000 steps, values of one sign: a state formed with a rounded 1 - s would be off by up to 3% of 1 / s."""
    from machinelearning_b200 import gated_scan
    T = 20000
    gate = torch.full((1, T, 2), -13.8, device="cuda")
    value = torch.ones(1, T, 2, device="cuda")
    h, last = gated_scan.gated_scan(gate, value)
    s = 1 / (1 + np.exp(np.float64(np.float32(13.8))))
    want = 1 - (1 - s) ** np.arange(1, T + 1)
    # every step: 2^-21 of s, and the step's rounding, at most half a unit of h (h up to 0.02)
    assert (np.abs(h[0, :, 0].double().cpu().numpy() - want) <= want * 2.0**-21 + 2.0**-24 * 2.0**-5 * np.arange(1, T + 1)).all()
    assert torch.equal(last[0], h[0, -1])


@pytest.mark.gpu
def test_strided_inputs_are_read_where_they_lie():
    from machinelearning_b200 import gated_scan
    gate, value, state, _, _, _, _ = _inputs(4, 50, 24, torch.float16)
    want = gated_scan.gated_scan(gate, value, state)
    time_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(4, 50, 61, device="cuda", dtype=torch.float16)
    odd = wide[..., 3:27]                                         # rows that begin between pairs
    odd.copy_(value)
    channels_first = gate.transpose(1, 2).contiguous().transpose(1, 2)
    for z, v in ((time_first(gate), value), (gate, odd), (channels_first, time_first(value))):
        got = gated_scan.gated_scan(z, v, state)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = gate[:, :1].expand(4, 50, 24)
    got, same = gated_scan.gated_scan(one, value), gated_scan.gated_scan(one.contiguous(), value)
    assert torch.equal(got[0], same[0])
    guarded = gated_scan.gated_scan(gate, value, state.to(torch.bfloat16))       # a state of another type
    assert torch.equal(guarded[1], gated_scan.gated_scan(gate, value, state.to(torch.bfloat16).float())[1])


@pytest.mark.gpu
def test_graph_capture_and_side_stream():
    from machinelearning_b200 import gated_scan
    gate, value, state, reset, lengths, dh, dlast = _inputs(2, 700, 64, torch.bfloat16)
    leaves = [t.detach().clone().requires_grad_() for t in (gate, value, state)]

    def step():
        h, last = gated_scan.gated_scan(*leaves, reset=reset, lengths=lengths)
        return h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (dh, dlast))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    del on_side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for scale in (1.0, 0.5):                                      # replayed on other values, beside an eager call
        with torch.no_grad():
            leaves[1].mul_(scale)
        graph.replay()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_compiled_caller_keeps_one_graph():
    from machinelearning_b200 import flash_cuda, gated_scan
    assert flash_cuda.is_available()
    gate, value, state, reset, _, dh, dlast = _inputs(2, 40, 32, torch.bfloat16)

    def call(z, v, s):
        h, last = gated_scan.gated_scan(z, v, s, activation="positive", reset=reset)
        return h * 2, last
    leaves = [t.detach().requires_grad_() for t in (gate, value, state)]
    want = call(*leaves)
    wanted = torch.autograd.grad(want, leaves, (dh, dlast))
    got = torch.compile(call, fullgraph=True)(*leaves)
    grads = torch.autograd.grad(got, leaves, (dh, dlast))
    assert all(torch.equal(a, b) for a, b in zip((*got, *grads), (*want, *wanted)))


@pytest.mark.gpu
def test_saved_tensors_that_change_raise_and_second_derivatives_raise():
    from machinelearning_b200 import gated_scan
    gate, value, state, _, _, dh, dlast = _inputs(1, 20, 8, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (gate, value, state)]
    z = leaves[0] * 1
    h, last = gated_scan.gated_scan(z, leaves[1], leaves[2])
    with torch.no_grad():
        z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad((h, last), leaves, (dh, dlast))
    h, last = gated_scan.gated_scan(*leaves)
    up = dh.detach().requires_grad_()
    (dz,) = torch.autograd.grad(h, leaves[0], up, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dz.sum().backward()


@pytest.mark.gpu
def test_refusals_on_the_device():
    from machinelearning_b200 import gated_scan
    z = torch.randn(2, 5, 8, device="cuda")
    for bad in ((z, z.half()), (z, z[:, :4]), (z[0], z[0]), (z.double(), z.double()), (z, z, z[:, 0, :4]), (z, z, z[:, 0].cpu())):
        with pytest.raises(ValueError, match="unsupported inputs"):
            gated_scan.gated_scan(*bad)
    for kw in ({"reset": torch.zeros(2, 5, device="cuda")}, {"reset": torch.zeros(2, 4, device="cuda", dtype=torch.bool)},
               {"lengths": torch.zeros(2, device="cuda")}, {"lengths": torch.zeros(3, device="cuda", dtype=torch.int32)}):
        with pytest.raises(ValueError, match="unsupported inputs"):
            gated_scan.gated_scan(z, z, **kw)
