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
