"""Norm and clip of many gradients: the oracle against torch, the refusals, and -- on the GPU -- against the oracle.

The norm: eights in float32 (8 2^-24 relative at most), everything else in float64, one rounding: within 2^-20; the factor adds 2^-22, and
an element its own rounding (u of its type; float32 results of 16-bit gradients: 2^-24).
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import step_f64

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
_id = lambda d: str(d).split(".")[-1]


def test_oracle_matches_torch():
    g = torch.Generator().manual_seed(0)
    for norm in (2.0, float("inf")):
        for limit in (0.5, 1e3):
            ps = [torch.nn.Parameter(torch.zeros(s, dtype=torch.float64)) for s in ((3, 4), (5,), ())]
            for p in ps:
                p.grad = torch.randn(p.shape, generator=g, dtype=torch.float64)
            total, want = step_f64.clip([p.grad.numpy().copy() for p in ps], limit, norm)
            assert abs(float(torch.nn.utils.clip_grad_norm_(ps, limit, norm)) - total) <= 1e-12
            assert all(np.abs(p.grad.numpy() - w).max() <= 1e-12 for p, w in zip(ps, want))


def test_entry_points_refuse_bad_arguments_before_any_launch():
    from machinelearning_b200 import _build, _lib
    _build.build()
    lib = _lib.load()
    class Grad(ctypes.Structure):
        _fields_ = [("grad", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_longlong), ("dtype", ctypes.c_int),
                    ("out_dtype", ctypes.c_int)]
    need = lib.nlfa_clip_scratch_bytes()
    def call(count=1, norm=2, total=256, s=256, sb=need, **g):
        a = (Grad * 1)(Grad(**{**dict(grad=256, out=None, n=8, dtype=2, out_dtype=0), **g}))
        return lib.nlfa_clip_grads(ctypes.addressof(a), count, 1.0, norm, 1, total, s, sb, None)
    assert call(count=-1) == 14 and call(norm=1) == 14
    assert call(total=None) == 1 and call(s=None) == 1 and call(grad=None) == 1
    assert call(s=264) == 6 and call(sb=need - 1) == 11 and call(total=258) == 6
    assert call(dtype=5) == 3 and call(out=512, out_dtype=7) == 3 and call(n=0) == 2
    assert call(grad=257) == 6 and call(out=514, out_dtype=0) == 6
    assert lib.nlfa_clip_grads(None, 1, 1.0, 2, 1, 256, 256, need, None) == 1


def test_python_call_refuses_what_it_does_not_take():
    from machinelearning_b200 import grad_clip
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(grad_clip.clip_grad_norm_([p], 1.0)) == 0.0     # no gradients, as torch
    assert float(grad_clip.grad_norm([])) == 0.0
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="CUDA"):
        grad_clip.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        grad_clip.clip_grad_norm_([p], 1.0, norm_type=1.0)


SHAPES = [(1,), (768,), (8193,), (333, 77), (), (16384,), (5, 7, 11), (100003,), (2,)]


def _params(shapes, dtypes, seed=0, size=1e-2, skew=0):
    """Parameters whose gradients lie in one buffer per type, `skew` elements off a 16-byte border."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps = []
    for i, s in enumerate(shapes):
        n = int(np.prod(s))
        dt = dtypes[i % len(dtypes)]
        store = torch.empty(n + 16, device="cuda", dtype=dt)
        store[skew:skew + n] = torch.randn(n, device="cuda", generator=g) * size * (1 + i % 3)
        p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dt))
        p.grad = store[skew:skew + n].view(s)
        ps.append(p)
    return ps


def _check(before, after, total, limit, norm=2.0):
    want_total, want = step_f64.clip([b.double().cpu().numpy() for b in before], limit, norm)
    assert abs(float(total) - want_total) <= 2.0**-20 * want_total
    for b, a, w in zip(before, after, want):
        a = a.double().cpu().numpy()
        tiny = 2.0**-25 if after[0].dtype == torch.float16 else 0.0
        # (a norm next to the limit may fall on either side of it: the factor is one to within the norm's bound)
        bound = (HALF_STEP[torch.float32] + 2.0**-19) * np.abs(w)
        bound = bound + (np.abs(w) * 2.0**-8 if torch.bfloat16 in (b.dtype,) else np.abs(w) * 2.0**-11 + 2.0**-25 if b.dtype == torch.float16 else 0.0)
        assert (np.abs(a - w) <= bound + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [2.0, float("inf")])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.float16], [torch.bfloat16], [torch.float32, torch.bfloat16, torch.float16]],
                         ids=lambda d: "-".join(map(_id, d)))
@pytest.mark.parametrize("skew", [0, 1, 8])
def test_norm_and_clip(dtypes, norm, skew):
    from machinelearning_b200 import grad_clip
    for limit in (0.01, 1e4):
        ps = _params(SHAPES, dtypes, skew=skew)
        before = [p.grad.clone() for p in ps]
        version = ps[1].grad._version
        total = grad_clip.clip_grad_norm_(ps, limit, norm)
        assert total.dtype == torch.float32 and total.shape == () and ps[1].grad._version > version
        _check(before, [p.grad for p in ps], total, limit, norm)
        if limit == 1e4:
            assert all(torch.equal(b, p.grad) for b, p in zip(before, ps))
        assert torch.equal(total, grad_clip.grad_norm(before, norm))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=_id)
def test_clip_into_other_tensors(dtype):
    from machinelearning_b200 import grad_clip
    for limit in (0.01, 1e4):
        ps = _params(SHAPES, [dtype])
        before = [p.grad.clone() for p in ps]
        store = [torch.full((p.grad.numel() + 5,), 7.0, device="cuda") for p in ps]
        outs = [s[i % 4:i % 4 + p.grad.numel()].view(p.shape) for i, (s, p) in enumerate(zip(store, ps))]    # also misaligned
        total = grad_clip.clip_grad_norm_(ps, limit, out=outs)
        assert all(torch.equal(b, p.grad) for b, p in zip(before, ps))
        want_total, want = step_f64.clip([b.double().cpu().numpy() for b in before], limit)
        assert abs(float(total) - want_total) <= 2.0**-20 * want_total
        for i, (o, w, s) in enumerate(zip(outs, want, store)):
            assert (np.abs(o.double().cpu().numpy() - w) <= 2.0**-18 * np.abs(w)).all()
            assert bool((s[:i % 4] == 7).all()) and bool((s[i % 4 + o.numel():] == 7).all())
        own = [p.grad for p in ps]                               # a gradient may be its own out
        again = grad_clip.clip_grad_norm_(ps, limit, out=own)
        assert torch.equal(again, total)
        _check(before, own, again, limit)


@pytest.mark.gpu
def test_many_tensors_and_large_ones():
    """More tensors than one launch takes; a piece count beyond the grid; an empty gradient among them."""
    from machinelearning_b200 import grad_clip
    for count in (47, 49, 320, 321, 2300):
        ps = _params([(1 + 37 * i % 500,) for i in range(count)], [torch.float32, torch.bfloat16])
        ps[3] = torch.nn.Parameter(torch.empty(0, device="cuda"))
        ps[3].grad = torch.empty(0, device="cuda")
        before = [p.grad.clone() for p in ps]
        total = grad_clip.clip_grad_norm_(ps, 0.05)
        _check(before, [p.grad for p in ps], total, 0.05)
    ps = _params([(9_000_001,), (3,)], [torch.float32])
    before = [p.grad.clone() for p in ps]
    total = grad_clip.clip_grad_norm_(ps, 1.0)
    _check(before, [p.grad for p in ps], total, 1.0)


@pytest.mark.gpu
def test_values_beyond_the_squares_range_and_not_finite():
    from machinelearning_b200 import grad_clip
    dev = dict(device="cuda")
    for value in (1e25, 1e-25, 3e38):
        x = torch.full((1000,), value, **dev)
        x[::7] = 0.0
        want = (x.double() ** 2).sum().sqrt()
        got = grad_clip.grad_norm([x])
        assert abs(float(got) - float(want.float())) <= 2.0**-22 * float(want) or (float(want) > 3.4e38 and torch.isinf(got))
        assert float(grad_clip.grad_norm([x], float("inf"))) == float(x.abs().max())
    for bad in (float("nan"), float("inf")):
        for norm in (2.0, float("inf")):
            p, q = torch.nn.Parameter(torch.zeros(100, **dev)), torch.nn.Parameter(torch.zeros(9000, **dev))
            p.grad, q.grad = torch.ones(100, **dev), torch.ones(9000, **dev)
            q.grad[8500] = bad
            want = torch.nn.utils.clip_grad_norm_([torch.nn.Parameter(t.clone()) for t in (p, q)], 1.0)
            ref = [torch.nn.Parameter(torch.zeros(100, **dev)), torch.nn.Parameter(torch.zeros(9000, **dev))]
            ref[0].grad, ref[1].grad = p.grad.clone(), q.grad.clone()
            want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm)
            with pytest.raises(RuntimeError, match="non-finite"):
                grad_clip.clip_grad_norm_([p, q], 1.0, norm, error_if_nonfinite=True)
            assert bool((p.grad == 1).all())
            got = grad_clip.clip_grad_norm_([p, q], 1.0, norm)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
            for a, b in zip((p, q), ref):
                assert torch.equal(a.grad.isnan(), b.grad.isnan()) and torch.equal(a.grad.nan_to_num(), b.grad.nan_to_num())


@pytest.mark.gpu
def test_layouts_and_refusals():
    from machinelearning_b200 import grad_clip
    g = torch.Generator(device="cuda").manual_seed(0)
    p, q, r = (torch.nn.Parameter(torch.zeros(6, 8, device="cuda")) for _ in range(3))
    wide = torch.randn(6, 20, device="cuda", generator=g)
    p.grad = torch.randn(8, 6, device="cuda", generator=g).t()   # column by column
    q.grad = wide[:, 3:11]                                       # with gaps
    rest = wide.clone()
    before = [p.grad.clone(), q.grad.clone()]
    total = grad_clip.clip_grad_norm_([p, q, r], 0.1)            # (r has no gradient)
    _check(before, [p.grad, q.grad], total, 0.1)
    assert torch.equal(wide[:, :3], rest[:, :3]) and torch.equal(wide[:, 11:], rest[:, 11:])
    with pytest.raises(ValueError, match="share memory"):
        grad_clip.clip_grad_norm_([p, p], 0.1)
    shared = torch.nn.Parameter(torch.zeros(6, 4, device="cuda"))
    shared.grad = p.grad[:, :4]                                  # half of p's
    with pytest.raises(ValueError, match="share memory"):
        grad_clip.clip_grad_norm_([p, shared], 0.1)
    assert float(grad_clip.grad_norm([p.grad, p.grad])) > float(grad_clip.grad_norm([p.grad]))     # reading twice is fine
    one = torch.nn.Parameter(torch.zeros(6, 8, device="cuda"))
    one.grad = torch.ones(6, 1, device="cuda").expand(6, 8)
    with pytest.raises(ValueError, match="share memory"):
        grad_clip.clip_grad_norm_([one], 0.1)
    assert abs(float(grad_clip.grad_norm([one.grad])) - 48**0.5) <= 1e-5
    d = torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=torch.float64))
    d.grad = torch.ones(3, device="cuda", dtype=torch.float64)
    with pytest.raises(ValueError, match="float32"):
        grad_clip.clip_grad_norm_([p, d], 0.1)
    with pytest.raises(ValueError, match="out"):
        grad_clip.clip_grad_norm_([p], 0.1, out=[torch.zeros(5, 8, device="cuda")])
    with pytest.raises(ValueError, match="0 tensors for 1"):
        grad_clip.clip_grad_norm_([p], 0.1, out=[])
    with pytest.raises(TypeError, match="must be a tensor"):
        grad_clip.clip_grad_norm_([p, 3.0], 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        grad_clip.grad_norm([torch.ones(3)])
    with pytest.raises(ValueError, match="share memory"):
        grad_clip.clip_grad_norm_([p, one], 0.1, out=[torch.zeros(6, 8, device="cuda"), p.grad])


@pytest.mark.gpu
def test_gradients_with_gaps_that_share_memory():
    """Refused as dense ones are; gradients that lie in one another's gaps are taken."""
    from machinelearning_b200 import grad_clip

    def clip(*views):
        ps = [torch.nn.Parameter(torch.zeros(v.shape, device="cuda")) for v in views]
        for p, v in zip(ps, views):
            p.grad = v
        return grad_clip.clip_grad_norm_(ps, 0.1)

    wide = torch.randn(6, 20, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    rest = wide.clone()
    left = wide[:, 3:11]
    for views in ((left, left), (left, wide[:, 10:15]), (wide[:, 12:], left, wide[4]), (wide[2, 3:5], left), (wide[:, ::2], wide[:, ::3]),
                  (wide[:, :, 1], wide[3, 7:8])):
        with pytest.raises(ValueError, match="share memory"):
            clip(*views)
    assert torch.equal(wide, rest)
    for views in ((left, wide[:, 11:], wide[:, :3]), (wide[:, ::2], wide[:, 1::2]), (wide[2, 11:15], left, wide[5, 11]),
                  (wide[..., 0], wide[..., 2], wide[..., 3])):
        before = [v.clone() for v in views]
        total = clip(*views)
        _check(before, views, total, 0.1)
        wide.copy_(rest)


@pytest.mark.gpu
def test_reproducible_captured_and_on_another_stream():
    from machinelearning_b200 import grad_clip
    ps = _params([(300, 400), (4097,), (9,)], [torch.float32])
    kept = [p.grad.clone() for p in ps]

    def step():
        for p, k in zip(ps, kept):
            p.grad.copy_(k)
        return grad_clip.clip_grad_norm_(ps, 0.5)
    total = step()
    want = [total.clone(), *(p.grad.clone() for p in ps)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        total = step()
        got = [total, *(p.grad.clone() for p in ps)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = step()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, [total, *(p.grad for p in ps)]))
    for k in kept:
        k.mul_(1e-3)
    graph.replay()                                               # within the limit now
    assert all(torch.equal(k, p.grad) for k, p in zip(kept, ps))
