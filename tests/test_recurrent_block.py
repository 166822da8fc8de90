"""The recurrent model: gated recurrence and gated feed-forward layer together, as ``whole_model`` calls them -- training against the same
model in tensor operations, decoding from states, and the captured step.
"""
import pytest
import torch

from machinelearning_b200 import whole_model as wm


def _shape(**kw):
    return wm.ModelShape(n_layer=2, d_model=96, n_head=3, head_dim=32, vocab_size=211, block_size=70, mixer="mingru", zero_init_proj=False, **kw)


def _model(device, seed=0, **kw):
    torch.manual_seed(seed)
    return wm.GPT(_shape(**kw)).to(device)


def test_plain_scan_is_the_recurrence():
    g = torch.Generator().manual_seed(0)
    z, v, s = torch.randn(3, 13, 5, generator=g), torch.randn(3, 13, 5, generator=g), torch.randn(3, 5, generator=g)
    reset, lengths = torch.rand(3, 13, generator=g) < 0.2, torch.tensor([13, 4, 0])
    h, last = wm.plain_scan(z, v, s, reset, lengths)
    f = torch.where(v < 0, torch.sigmoid(v), v + 0.5)
    for b in range(3):
        at = s[b]
        for t in range(13):
            if t >= lengths[b]:
                assert bool((h[b, t] == 0).all())
                continue
            at = torch.where(reset[b, t], torch.zeros(5), at)
            at = (1 - torch.sigmoid(z[b, t])) * at + torch.sigmoid(z[b, t]) * f[b, t]
            assert float((h[b, t] - at).abs().max()) <= 2.0**-20
        assert float((last[b] - at).abs().max()) <= 2.0**-20


def test_model_on_the_cpu():
    """Flags are inert without a device; every parameter has a gradient; chunks from states are the whole."""
    model = _model("cpu", fused_ffn=True, fused_scan=True)
    idx = torch.randint(0, 211, (2, 70), generator=torch.Generator().manual_seed(1))
    logits, loss = model(idx, idx)
    loss.backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())
    assert model.flops_per_token() == 6.0 * model.n_params()
    states = None
    for a, b in ((0, 1), (1, 2), (2, 40), (40, 70)):
        out, states = model.forward_states(idx[:, a:b], states)
        assert float((out - logits[:, b - 1]).detach().abs().max()) <= 1e-5
    with pytest.raises(ValueError, match="recurrent"):
        wm.GPT(wm.ModelShape(n_layer=1, d_model=64, n_head=2, head_dim=32, vocab_size=50)).forward_states(idx)
    with pytest.raises(ValueError, match="mixer"):
        wm.ModelShape(mixer="lstm")


@pytest.mark.gpu
def test_training_matches_the_plain_model():
    """float32: both sides' sums are off by up to some 2^-20 of their magnitudes, layer by layer."""
    plain, fused = _model("cuda"), _model("cuda", fused_ffn=True, fused_scan=True, fused_embedding=True, fused_loss=True)
    idx = torch.randint(0, 211, (5, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    _, want = plain(idx, idx)
    _, got = fused(idx, idx)
    want.backward()
    got.backward()
    assert abs(float(got.detach()) - float(want.detach())) <= 2.0**-17 * float(want.detach())
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        assert float((q.grad - p.grad).norm()) <= 2.0**-15 * float(p.grad.norm()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decoding_from_states(dtype):
    """Prefill of a padded batch, then token by token: the logits of the whole sequences."""
    model = _model("cuda", fused_ffn=True, fused_scan=True, fused_embedding=True)
    idx = torch.randint(0, 211, (3, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    lengths = torch.tensor([40, 1, 23], device="cuda")
    # Both ways compute the same products; in bf16 they round the same values apart from where a sum's last bit tips a rounding: some steps of 2^-8
    most = 2.0**-15 if dtype == torch.float32 else 2.0**-4
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype, enabled=dtype != torch.float32):
        out, states = model.forward_states(idx[:, :40], lengths=lengths)
        at = lengths.clone()
        for _ in range(6):
            for b in range(3):
                whole, _ = model(idx[b:b + 1, :int(at[b])])
                scale = float(whole.float().abs().max())
                assert float((out[b].float() - whole[0, -1].float()).abs().max()) <= most * scale
            out, states = model.forward_states(idx.gather(1, at[:, None]), states)
            at += 1


@pytest.mark.gpu
def test_captured_step_and_decoding_beside_it():
    """DataParallelStep with every fused part, captured: its replays and the eager step give the same losses; decoding runs between them."""
    idx = torch.randint(0, 211, (4, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    losses = []
    for captured in (False, True):
        model = _model("cuda", fused_ffn=True, fused_scan=True, fused_embedding=True, fused_loss=True)
        step = wm.DataParallelStep(model, lr=1e-3, fused_clip=True)
        if captured:
            step.capture(idx, idx)
        seen = []
        for i in range(3):
            seen.append(float(step.step(idx.roll(i, 1), idx)))
            with torch.autocast("cuda", dtype=torch.bfloat16):
                out, _ = model.forward_states(idx)
            assert bool(torch.isfinite(out).all())
        losses.append(seen)
        step.close()
    assert losses[0] == losses[1]


@pytest.mark.gpu
def test_calls_on_two_streams_and_a_backward_that_runs_twice():
    """Workspaces are each call's own: calls that overlap, and a graph that is kept, give the bits of calls alone."""
    from machinelearning_b200 import gated_ffn, gated_scan
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, wg, wu, wd = (t.bfloat16().requires_grad_() for t in (rand(900, 128), rand(320, 128) * 0.1, rand(320, 128) * 0.1, rand(128, 320) * 0.1))
    z, v, s = (t.requires_grad_() for t in (rand(2, 3000, 40), rand(2, 3000, 40), rand(2, 40)))

    def both():
        y = gated_ffn.gated_ffn(x, wg, wu, wd)
        h, last = gated_scan.gated_scan(z, v, s)
        return y, h, last

    def grads(out, keep=False):
        y, h, last = out
        return (*torch.autograd.grad(y, (x, wg, wu, wd), torch.ones_like(y), retain_graph=keep),
                *torch.autograd.grad((h, last), (z, v, s), (torch.ones_like(h), torch.ones_like(last)), retain_graph=keep))
    out = both()
    want = (*out, *grads(out, keep=True))
    assert all(torch.equal(a, b) for a, b in zip(grads(out), want[3:]))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for st in streams:
        with torch.cuda.stream(st):
            out = both()
            got.append((*out, *grads(out)))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


@pytest.mark.gpu
def test_outputs_have_no_more_than_their_own_memory():
    """Results between guard values: nothing behind the last row or column is written."""
    from machinelearning_b200 import _lib, flash_cuda, gated_scan
    lib = flash_cuda._load()
    g = torch.Generator(device="cuda").manual_seed(6)
    for B, T, D in ((2, 37, 24), (1, 1030, 7), (3, 20, 72)):
        z, v = torch.randn(B, T, D, device="cuda", generator=g), torch.randn(B, T, D, device="cuda", generator=g)
        guarded = torch.full((B * T * D + 128,), 777.0, device="cuda")
        last = torch.full((B * D + 64,), 777.0, device="cuda")
        scratch = gated_scan._scratch(lib, z)
        st = lib.nlfa_gated_scan_fwd(z.data_ptr(), T * D, D, v.data_ptr(), T * D, D, 0, None, None, None, 0, 0, B, T, D, guarded[64:].data_ptr(),
                                     last[32:].data_ptr(), None, 0, scratch.data_ptr(), scratch.numel(), torch.cuda.current_stream().cuda_stream)
        assert st == _lib.OK
        want = gated_scan.gated_scan(z, v)
        assert torch.equal(guarded[64:-64].view(B, T, D), want[0]) and torch.equal(last[32:-32].view(B, D), want[1])
        assert bool((guarded[:64] == 777).all()) and bool((guarded[-64:] == 777).all()) and bool((last[:32] == 777).all()) and bool((last[-32:] == 777).all())
    for n, d, F, o in ((70, 64, 128, 72), (9, 24, 40, 19), (300, 100, 70, 130)):
        x, wg, wu, wd = (torch.randn(*s, device="cuda", generator=g) for s in ((n, d), (F, d), (F, d), (o, F)))
        y = torch.full((n * o + 128,), 777.0, device="cuda")
        copies = lib.nlfa_gated_ffn_copies(x.data_ptr(), 0, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), 0, 0, n, d, F, 1)
        tape = torch.empty(lib.nlfa_gated_ffn_tape_bytes(n, d, F, o, 0, copies, 1), dtype=torch.uint8, device="cuda")
        scratch = torch.empty(lib.nlfa_gated_ffn_scratch_bytes(n, d, F, o, 0, copies, 1, 0), dtype=torch.uint8, device="cuda")
        at = torch.cuda.current_stream().cuda_stream
        assert lib.nlfa_gated_ffn_fwd(x.data_ptr(), 0, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), 0, 0, 0, n, d, F, o, y[64:].data_ptr(), copies, 1,
                                      tape.data_ptr(), tape.numel(), scratch.data_ptr(), scratch.numel(), at) == _lib.OK
        out = [torch.full((a * b + 128,), 777.0, device="cuda") for a, b in ((n, d), (F, d), (F, d), (o, F))]
        back = torch.empty(lib.nlfa_gated_ffn_scratch_bytes(n, d, F, o, 0, copies, 1, 1), dtype=torch.uint8, device="cuda")
        dy = torch.randn(n, o, device="cuda", generator=g)
        assert lib.nlfa_gated_ffn_bwd(dy.data_ptr(), None, 0, None, None, None, 0, 0, 0, n, d, F, o, copies, tape.data_ptr(), tape.numel(),
                                      *(t[64:].data_ptr() for t in out), back.data_ptr(), back.numel(), at) == _lib.OK
        for t in (y, *out):
            assert bool((t[:64] == 777).all()) and bool((t[-64:] == 777).all()) and not bool((t[64:-64] == 777).any())


@pytest.mark.gpu
def test_rows_behind_two_to_the_31_elements():
    """What stands at the end of tensors of more than 2^31 elements is what a short call of the same rows gives, up to where sums are cut.

    Two float32 sums of one value round to neighbours in bfloat16 at most: 2^-7 of it, beside the sums' own difference.  Recurrence: states and gradients
    below 16, 2^-22 of which a walk is off by: 2^-18.  Layer: 2^-17 of the summands' magnitudes for each of the two calls (tests of the layer), which are below 64
    for y (2,048 of some 0.4 x 0.018) and below 512 for dx (twice 2,048 of some 0.5 x 0.1)."""
    from machinelearning_b200 import gated_ffn, gated_scan
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s, std=1.0: (torch.randn(*s, device="cuda", dtype=torch.bfloat16, generator=g) * std).requires_grad_()

    def close(got, want, beside):
        want = want.float()
        assert bool(((got.float() - want).abs() <= 2.0**-7 * want.abs() + beside).all())

    for width in (1032, 1031):
        gate, value, dh = (rand(2, 1 << 20, width) for _ in range(3))
        h, last = gated_scan.gated_scan(gate, value)
        grads = torch.autograd.grad(h, (gate, value), dh)
        short = [t.detach()[1:, -4096:].clone().requires_grad_() for t in (gate, value)]
        end, end_last = gated_scan.gated_scan(*short)
        want = torch.autograd.grad(end, short, dh.detach()[1:, -4096:])
        # (behind 1,000 steps nothing of the state in front of them is left)
        for a, b in zip((h, *grads), (end, *want)):
            close(a.detach()[1:, -3096:], b.detach()[:, 1000:], 2.0**-18)
        close(last.detach()[1:], end_last.detach(), 2.0**-18)
        del gate, value, dh, h, last, grads, short, end, want
        torch.cuda.empty_cache()
    n = 1_100_000
    x, wg, wu, wd, dy = rand(n, 64), rand(2048, 64, std=0.125), rand(2048, 64, std=0.125), rand(64, 2048, std=2048**-0.5), rand(n, 64)
    y = gated_ffn.gated_ffn(x, wg, wu, wd)
    dx = torch.autograd.grad(y, x, dy)[0]
    for at in (n // 2, n - 700):
        some = x.detach()[at:at + 700].clone().requires_grad_()
        part = gated_ffn.gated_ffn(some, wg, wu, wd)
        close(y.detach()[at:at + 700], part.detach(), 2.0**-16 * 64)
        close(dx[at:at + 700], torch.autograd.grad(part, some, dy.detach()[at:at + 700])[0], 2.0**-16 * 512)
    del x, y, dy, dx
    torch.cuda.empty_cache()
