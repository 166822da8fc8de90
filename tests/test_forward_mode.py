"""Tensors that carry a forward-mode tangent: no operator has a rule for one, so each refuses them instead of giving a result without a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def test_tangents_are_told_from_plain_tensors():
    from machinelearning_b200 import flash_cuda
    x, y = torch.randn(3), torch.randn(3)
    flash_cuda.refuse_tangents("op", x, None, y)
    with fwad.dual_level():
        flash_cuda.refuse_tangents("op", x, None, y)
        dual = fwad.make_dual(x, y)
        for args in ((dual,), (y, None, dual)):
            with pytest.raises(ValueError, match="op: forward-mode"):
                flash_cuda.refuse_tangents("op", *args)
    flash_cuda.refuse_tangents("op", x)


def _calls():
    from machinelearning_b200 import flash_cuda, gated_ffn, gated_scan, head_loss, qk_prologue, token_embedding, value_gate
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g, dtype=torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.long, device="cuda")
    return {
        "gated_ffn": (gated_ffn.gated_ffn, [rand(4, 64), rand(64, 64), rand(64, 64), rand(64, 64)]),
        "gated_scan": (lambda z, v, s: gated_scan.gated_scan(z, v, s)[0], [rand(2, 5, 8), rand(2, 5, 8), rand(2, 8).float()]),
        "flash_attn": (flash_cuda.flash_attn, [rand(1, 16, 2, 64), rand(1, 16, 2, 64), rand(1, 16, 2, 64)]),
        "flash_attn_cached": (flash_cuda.flash_attn_cached, [rand(1, 16, 2, 64), rand(1, 2, 16, 64), rand(1, 2, 16, 64)]),
        "qk_prologue": (qk_prologue.qk_prologue, [rand(1, 16, 2, 64), rand(64)]),
        "value_blend": (value_gate.value_blend, [rand(1, 16, 2, 64), rand(1, 16, 2, 64), rand(1).float()]),
        "head_gate": (value_gate.head_gate, [rand(1, 16, 2, 64), rand(1, 16, 2)]),
        "linear_cross_entropy": (lambda x, w: head_loss.linear_cross_entropy(x, w, ids), [rand(4, 64), rand(100, 64)]),
        "embedding": (lambda w: token_embedding.embedding(ids, w), [rand(100, 64)]),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gated_ffn", "gated_scan", "flash_attn", "flash_attn_cached", "qk_prologue", "value_blend", "head_gate",
                                  "linear_cross_entropy", "embedding"])
def test_operators_refuse_tangents(name):
    from machinelearning_b200 import flash_cuda
    assert flash_cuda.is_available()
    call, args = _calls()[name]
    want = call(*args)
    for needs in (False, True):                                    # with reverse mode beside it as well
        with fwad.dual_level():
            assert torch.equal(call(*args), want)                  # a level alone changes nothing
            for i, t in enumerate(args):
                leaf = t.detach().requires_grad_(needs)
                dual = fwad.make_dual(leaf, torch.ones_like(t))
                with pytest.raises(ValueError, match=f"{name}: forward-mode"):
                    call(*args[:i], dual, *args[i + 1:])
    assert torch.equal(call(*args), want)
