"""The ends of a training step together, as the whole-model caller uses them: embedding, head with its loss, clip."""
import pytest
import torch

from machinelearning_b200 import whole_model as wm

SHAPE = dict(n_layer=2, d_model=128, n_head=2, head_dim=64, vocab_size=515, block_size=96)


def test_on_the_cpu_the_flags_change_nothing():
    """The kernels do not take CPU tensors: torch's own lines run, logits and all."""
    x, y = wm.synthetic_tokens(515, 2, 96)
    losses = []
    for on in (False, True):
        torch.manual_seed(0)
        model = wm.GPT(wm.ModelShape(**SHAPE, fused_loss=on, fused_embedding=on))
        step = wm.DataParallelStep(model, dtype=torch.float32, fused_clip=on)
        logits, _ = model(x, y)
        assert logits is not None
        losses.append([float(step.step(x, y)) for _ in range(3)])
    assert losses[0] == losses[1]


def _model(on, **more):
    torch.manual_seed(0)
    model = wm.GPT(wm.ModelShape(**{**SHAPE, **more}, flash_cuda=True, zero_init_proj=False, fused_loss=on, fused_embedding=on)).cuda()
    return model


def _tokens():
    x, y = wm.synthetic_tokens(515, 3, 96, seed=1)
    y[0, 40:] = -1                                               # a padded row
    return x.cuda(), y.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [True, False])
def test_gradients_of_every_parameter(tied):
    """float32: every gradient of the model with its ends through the kernels equals the model's without them.  Both sides
    round to float32; sums over 288 tokens and 515 words in another order differ by under 2^-14 of a tensor's largest gradient
    (600 terms, 2^-24 each, through 2 layers whose products amplify a difference at their output at most 16 times)."""
    x, y = _tokens()
    grads = []
    for on in (False, True):
        model = _model(on, tie_embeddings=tied)
        logits, loss = model(x, y)
        assert (logits is None) == on
        loss.backward()
        grads.append((float(loss.detach()), {n: p.grad for n, p in model.named_parameters() if p.grad is not None}))
    assert abs(grads[0][0] - grads[1][0]) <= 2.0**-18 * grads[0][0]
    assert grads[0][1].keys() == grads[1][1].keys()
    for name, want in grads[0][1].items():
        got = grads[1][1][name]
        assert got.dtype == want.dtype
        assert float((got - want).abs().max()) <= 2.0**-14 * float(want.abs().max()), name


@pytest.mark.gpu
def test_steps_eager_and_captured():
    """Three steps under bf16 autocast with all three operators: the captured step gives the eager one's bits, loss and parameters."""
    x, y = _tokens()
    runs = []
    for captured in (False, True):
        model = _model(True)
        step = wm.DataParallelStep(model, fused_clip=True, grad_clip=0.05)
        if captured:
            step.capture(x, y)
        losses = [float(step.step(x, y)) for _ in range(3)]
        runs.append((losses, {n: p.detach().clone() for n, p in model.named_parameters()}))
        step.close()
    assert runs[0][0] == runs[1][0]
    assert all(torch.equal(runs[0][1][n], runs[1][1][n]) for n in runs[0][1])
    assert all(torch.isfinite(p).all() for p in runs[0][1].values())


@pytest.mark.gpu
def test_clip_of_the_step():
    """After a backward, the kernels' norm and clipped gradients are torch's to rounding (2^-18: torch adds norms of tensors in float32)."""
    from machinelearning_b200 import grad_clip
    x, y = _tokens()
    model = _model(True)
    model(x, y)[1].backward()
    want = [p.grad.clone() for p in model.parameters() if p.grad is not None]
    norm = grad_clip.grad_norm(want)
    limit = 0.3 * float(norm)
    ref = [torch.nn.Parameter(torch.empty_like(g)) for g in want]
    for p, g in zip(ref, want):
        p.grad = g.clone()
    total = torch.nn.utils.clip_grad_norm_(ref, limit)
    got = grad_clip.clip_grad_norm_(model.parameters(), limit)
    assert abs(float(got) - float(total)) <= 2.0**-18 * float(total) and torch.equal(got, norm)
    for a, p in zip(ref, (p for p in model.parameters() if p.grad is not None)):
        assert float((a.grad - p.grad).abs().max()) <= 2.0**-17 * float(a.grad.abs().max())


@pytest.mark.gpu
def test_two_streams_and_a_replay_at_once():
    """Calls that overlap on the GPU -- two streams, and a captured step replayed beside eager ones -- give each its own bits."""
    from machinelearning_b200 import grad_clip, head_loss, token_embedding

    def job(seed, n, V, d, dtype):
        g = torch.Generator(device="cuda").manual_seed(seed)
        table = torch.randn(V, d, device="cuda", generator=g).to(dtype).requires_grad_()
        idx, t = (torch.randint(0, V, (n,), device="cuda", generator=g) for _ in range(2))

        def step():
            x = token_embedding.embedding(idx, table, scale=0.2)
            loss = head_loss.linear_cross_entropy(x, table, t)
            (grad,) = torch.autograd.grad(loss, (table,))
            leaf = torch.nn.Parameter(torch.empty_like(table))
            leaf.grad = grad
            return loss.detach(), grad_clip.clip_grad_norm_([leaf], 1e-3), leaf.grad
        return step
    jobs = [job(1, 900, 3000, 192, torch.bfloat16), job(2, 700, 5000, 96, torch.float32), job(3, 40, 2000, 64, torch.float16)]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = jobs[2]()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[], []]
    for _ in range(8):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(jobs[k]())
        with torch.cuda.stream(streams[2]):
            graph.replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for one in got[k] for a, b in zip(one, want[k]))
    assert all(torch.equal(a, b) for a, b in zip(captured, want[2]))
