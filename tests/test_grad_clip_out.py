"""The clip into other tensors where gradients have gaps: an out that lies over one is refused, one in the gaps is taken."""
import pytest
import torch

from test_grad_clip import _check


def _parameters(*grads):
    ps = [torch.nn.Parameter(torch.zeros(g.shape, device="cuda", dtype=g.dtype)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


@pytest.mark.gpu
def test_out_over_a_gradient_with_gaps():
    from machinelearning_b200 import grad_clip
    buf = torch.randn(6, 20, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    rest, flat = buf.clone(), buf.view(-1)
    other = torch.randn(12, device="cuda")
    kept = other.clone()
    left = buf[:, :8]
    free = lambda t: torch.zeros(t.shape, device="cuda")
    # its own out over it, another's, another's that is that gradient itself, in one element only
    for grads, outs in (((left,), (flat[:48].view(6, 8),)), ((left, other), (free(left), flat[7:19])), ((left, buf[2]), (free(left), buf[2])),
                        ((buf[:, ::3], other), (buf.new_zeros(6, 7), flat[105:117])),
                        ((buf[:1, :8].expand(5, 8), other), (buf.new_zeros(5, 8), flat[4:16]))):
        with pytest.raises(ValueError, match="share memory"):
            grad_clip.clip_grad_norm_(_parameters(*grads), 0.1, out=list(outs))
    assert torch.equal(buf, rest) and torch.equal(other, kept)
    # beside it, in its gaps, and gradients that share memory with one another but with no out
    for grads, outs in (((left, other), (free(left), flat[8:20])), ((left, buf[:, 3:8], other), (free(left), free(buf[:, 3:8]), flat[48:60])),
                        ((buf[:1, :8].expand(5, 8),), (buf.new_zeros(5, 8),))):
        before = [g.clone() for g in grads]
        total = grad_clip.clip_grad_norm_(_parameters(*grads), 0.1, out=list(outs))
        _check(before, outs, total, 0.1)
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
        buf.copy_(rest)
