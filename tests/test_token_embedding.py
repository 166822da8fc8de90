"""Token embedding: the oracle against torch autograd in float64, the refusals, and -- on the GPU -- rows bit for bit and
the table's gradient against the oracle.

A gradient row is one float32 chain of its token's rows (or of runs of them, whose sums are added), scaled and rounded once: off by at most
(m + 2) 2^-24 of its summands' magnitudes for m rows, and half a step of the output's type (fp16 below its normal range: 2^-25).
"""
import numpy as np
import pytest
import torch

from oracle import step_f64

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
_id = lambda d: str(d).split(".")[-1]


def test_oracle_matches_autograd():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(7, 5, generator=g, dtype=torch.float64).requires_grad_()
    idx = torch.randint(0, 7, (40,), generator=g)
    up = torch.randn(40, 5, generator=g, dtype=torch.float64)
    (want,) = torch.autograd.grad(torch.nn.functional.embedding(idx, w, padding_idx=2) * 3.0, w, up)
    dw, _ = step_f64.embedding_backward(up.numpy(), idx.numpy(), 7, 3.0, 2)
    assert np.abs(dw - want.numpy()).max() <= 1e-13


def test_entry_points_refuse_bad_arguments_before_any_launch():
    from machinelearning_b200 import _build, _lib
    _build.build()
    lib = _lib.load()
    fwd = lambda ids=256, ib=8, w=256, dt=2, out=256, n=4, V=10, d=8: lib.nlfa_embedding_fwd(ids, ib, w, dt, out, n, V, d, 1.0, None)
    assert fwd(V=0) == 2 and fwd(d=0) == 2 and fwd(n=-1) == 2 and fwd(dt=4) == 3 and fwd(ib=2) == 14
    assert fwd(ids=None) == 1 and fwd(w=None) == 1 and fwd(out=None) == 1
    assert fwd(w=257) == 6 and fwd(out=258, dt=0) == 6 and fwd(ids=260) == 6
    assert fwd(n=0, ids=None, w=None, out=None) == 0
    need = lib.nlfa_embedding_scratch_bytes(4, 10, 8)
    assert need > 0 and lib.nlfa_embedding_scratch_bytes(4, 0, 8) == 0

    def bwd(g=256, dt=2, ids=256, ib=8, dw=256, n=4, V=10, d=8, s=256, sb=need):
        return lib.nlfa_embedding_bwd(g, dt, ids, ib, dw, n, V, d, 1.0, -1, s, sb, None)
    assert bwd(V=0) == 2 and bwd(dt=9) == 3 and bwd(ib=3) == 14
    assert bwd(g=None) == 1 and bwd(ids=None) == 1 and bwd(dw=None) == 1 and bwd(s=None) == 1
    assert bwd(s=264) == 6 and bwd(dw=257) == 6 and bwd(ids=260) == 6 and bwd(sb=need - 1) == 11


def test_python_call_refuses_what_it_does_not_take():
    from machinelearning_b200 import token_embedding
    w, idx = torch.randn(9, 8), torch.zeros(4, dtype=torch.long)
    assert not token_embedding.supports(idx, w)
    with pytest.raises(ValueError, match="unsupported inputs"):
        token_embedding.embedding(idx, w)
    with pytest.raises(ValueError, match="padding_idx"):
        token_embedding.embedding(idx, w, padding_idx=9)


def _check_gradient(dw, up, idx, rows, scale=1.0, padding=None):
    want, size = step_f64.embedding_backward(up.detach().double().cpu().reshape(-1, up.shape[-1]).numpy(), idx.cpu().reshape(-1).numpy(), rows,
                                             scale, padding)
    m = np.bincount(idx.cpu().reshape(-1).clamp(0, rows - 1).numpy(), minlength=rows)[:, None]
    bound = HALF_STEP[dw.dtype] * np.abs(want) + (m + 2) * 2.0**-24 * size * 1.01
    if dw.dtype == torch.float16:
        bound = bound + 2.0**-25
    assert (np.abs(dw.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=_id)
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 50304, 768), (17, 5, 3), (1000, 7, 130), (3001, 1009, 100), (5000, 70000, 36),
                                   (9000, 300, 520), (40000, 2, 64), (2500, 131073, 8)])
def test_rows_and_gradient(dtype, n, V, d):
    from machinelearning_b200 import token_embedding
    g = torch.Generator(device="cuda").manual_seed(n + V)
    w = torch.randn(V, d, device="cuda", generator=g).to(dtype).requires_grad_()
    # half of the positions on few tokens, so that some sums run over many runs of positions
    idx = torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, torch.randint(0, V, (n,), device="cuda", generator=g),
                      torch.randint(0, min(V, 3), (n,), device="cuda", generator=g))
    up = torch.randn(n, d, device="cuda", generator=g).to(dtype)
    for scale, padding in ((1.0, None), (d**0.5, 0)):
        out = token_embedding.embedding(idx, w, scale=scale, padding_idx=padding)
        assert torch.equal(out, (w.detach()[idx].float() * scale).to(dtype))
        (dw,) = torch.autograd.grad(out, w, up)
        _check_gradient(dw, up, idx, V, float(np.float32(scale)), padding)


@pytest.mark.gpu
def test_one_token_everywhere():
    """Every position the same token: its sum runs through all runs of positions, shared by a CTA's warps."""
    from machinelearning_b200 import token_embedding
    w = torch.zeros(400, 72, device="cuda", requires_grad=True)
    idx = torch.full((30, 1000), 123, device="cuda")
    up = torch.randn(30, 1000, 72, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    (dw,) = torch.autograd.grad(token_embedding.embedding(idx, w), w, up)
    _check_gradient(dw, up, idx, 400)
    assert int((dw != 0).any(1).sum()) == 1


@pytest.mark.gpu
def test_layouts_ids_outside_the_table_and_no_ids():
    from machinelearning_b200 import token_embedding
    g = torch.Generator(device="cuda").manual_seed(2)
    store = torch.randn(50 * 24 + 1, device="cuda", generator=g).half()
    w = store[1:].view(50, 24).requires_grad_()                  # 2 bytes off
    idx = torch.randint(0, 50, (6, 7), device="cuda", generator=g)
    idx[2, 3], idx[4, 4], idx[5, 5] = 50, -1, 1 << 40
    out = token_embedding.embedding(idx.t(), w)
    inside = (idx.t() >= 0) & (idx.t() < 50)
    assert out.shape == (7, 6, 24) and bool(torch.isnan(out[~inside]).all()) and torch.equal(out[inside], w.detach()[idx.t()[inside]])
    up = torch.randn(7, 6, 24, device="cuda", generator=g).half()
    up[~inside] = float("inf")                                   # reaches nothing
    (dw,) = torch.autograd.grad(out, w, up)
    _check_gradient(dw, up[inside], idx.t()[inside], 50)
    small = torch.where(inside, idx.t(), 0).int()                # int32, strided
    assert torch.equal(token_embedding.embedding(small, w), w.detach()[small.long()])
    (dw2,) = torch.autograd.grad(token_embedding.embedding(small, w).float().sum(), w)     # an expanded gradient
    _check_gradient(dw2, torch.ones(7, 6, 24, device="cuda"), small, 50)
    wt = w.detach().t().contiguous().t().requires_grad_()
    assert torch.equal(token_embedding.embedding(small, wt), w.detach()[small.long()])
    empty = token_embedding.embedding(idx[:0], w)
    assert empty.shape == (0, 7, 24)
    (dw,) = torch.autograd.grad(empty.sum(), w)
    assert bool((dw == 0).all())
    assert bool((token_embedding.embedding(idx, w, padding_idx=-1) == token_embedding.embedding(idx, w)).logical_or(torch.isnan(w.detach()[0, 0] * 0 + token_embedding.embedding(idx, w))).all())
    with pytest.raises(ValueError, match="unsupported inputs"):
        token_embedding.embedding(idx.float(), w)
    with pytest.raises(ValueError, match="unsupported inputs"):
        token_embedding.embedding(idx.cpu(), w)


@pytest.mark.gpu
def test_reproducible_captured_and_on_another_stream():
    from machinelearning_b200 import token_embedding
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(500, 136, device="cuda", generator=g).bfloat16().requires_grad_()
    idx = torch.randint(0, 500, (4000,), device="cuda", generator=g)
    idx[::3] = 11
    up = torch.randn(4000, 136, device="cuda", generator=g).bfloat16()

    def step():
        out = token_embedding.embedding(idx, w, scale=2.0)
        return out.detach(), torch.autograd.grad(out, w, up)[0]
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    kept = idx.clone()
    idx.copy_(torch.randint(0, 500, (4000,), device="cuda", generator=g))
    changed = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(changed, captured))
    idx.copy_(kept)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, captured))


@pytest.mark.gpu
def test_gradient_against_differences_and_no_second_derivative():
    from machinelearning_b200 import token_embedding
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(20, 16, device="cuda", generator=g).requires_grad_()
    idx = torch.randint(0, 20, (64,), device="cuda", generator=g)
    up, v = torch.randn(64, 16, device="cuda", generator=g), torch.randn(20, 16, device="cuda", generator=g)
    (dw,) = torch.autograd.grad(token_embedding.embedding(idx, w, scale=1.5), w, up)
    with torch.no_grad():                                        # linear: the difference is the derivative
        f = lambda t: float((token_embedding.embedding(idx, t, scale=1.5).double() * up.double()).sum())
        slope = (f(w + v) - f(w - v)) / 2
    assert abs(slope - float((dw.double() * v.double()).sum())) <= 1024 * 2.0**-22 * 8
    up.requires_grad_()
    (d,) = torch.autograd.grad(token_embedding.embedding(idx, w), w, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        d.sum().backward()


@pytest.mark.gpu
def test_compiled_caller_matches_eager():
    from machinelearning_b200 import flash_cuda, token_embedding
    assert flash_cuda.is_available()
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn(60, 64, device="cuda", generator=g).requires_grad_()
    idx = torch.randint(0, 60, (4, 25), device="cuda", generator=g)
    f = lambda i, t: (token_embedding.embedding(i, t, scale=8.0) ** 2).sum()
    want = torch.autograd.grad(f(idx, w), w)[0]
    assert torch.equal(torch.autograd.grad(torch.compile(f, fullgraph=True)(idx, w), w)[0], want)
