"""The table's gradient where the sort and the sums take other turns than at small sizes: runs of 32, 64 and 128 sorted positions, tokens
that begin and end at borders of 32, ids without a gradient in a later block of a run, three passes of the sort, wide digits in
CTAs of 1,024, rows of more slabs than a grid has along y.

Bounds as in test_token_embedding.py: (m + 2) 2^-24 of the summands' magnitudes for m rows of a token, and half a step of the type.
"""
import pytest
import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _run_length(n, d):
    """Positions of a warp, as the entry point chooses it (csrc/embedding.cu)."""
    run = 16
    while run < 128 and n * ((d + 127) // 128) // (2 * run) >= 64 * 148:
        run *= 2
    return run


def _check(idx, up, V, scale=1.0, padding=None, dtype=torch.float32):
    from machinelearning_b200 import token_embedding
    w = torch.zeros(V, up.shape[1], device="cuda", dtype=dtype, requires_grad=True)
    out = token_embedding.embedding(idx, w, scale=scale, padding_idx=padding)
    (dw,) = torch.autograd.grad(out, w, up)
    keep = (idx >= 0) & (idx < V)
    if padding is not None:
        keep &= idx != padding
    ids, rows = idx[keep].long(), up[keep].double() * scale
    # (index_add_ in 64 bits: its order does not show at these bounds)
    want = torch.zeros(V, up.shape[1], device="cuda", dtype=torch.float64).index_add_(0, ids, rows)
    size = torch.zeros_like(want).index_add_(0, ids, rows.abs())
    m = torch.bincount(ids, minlength=V)[:, None]
    bound = HALF_STEP[dtype] * want.abs() + (m + 2) * 2.0**-24 * size * 1.01 + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert bool(((dw.double() - want).abs() <= bound).all())
    assert bool((dw[m[:, 0] == 0] == 0).all())


def _rows(n, d, dtype=torch.float32, seed=0):
    return torch.randn(n, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,dtype,run", [(30000, 1000, torch.bfloat16, 16), (40000, 1000, torch.bfloat16, 32), (40000, 2000, torch.float32, 64),
                                           (90001, 1030, torch.float16, 64), (131072, 1024, torch.bfloat16, 64),
                                           (131072, 1290, torch.float32, 128), (400000, 700, torch.bfloat16, 128), (160001, 2056, torch.float32, 128)])
def test_longer_runs(n, d, dtype, run):
    """Tokens of 1 to 400 positions, so that in sorted order they begin and end anywhere: at borders of 32, of runs, and next to them."""
    assert _run_length(n, d) == run
    g = torch.Generator(device="cuda").manual_seed(n)
    V = 5000
    many = torch.tensor([1, 2, 31, 32, 33, 63, 64, 65, 96, 128, 129, 200, 400], device="cuda")
    ids = torch.repeat_interleave(torch.arange(V, device="cuda"), many[torch.randint(0, 13, (V,), device="cuda", generator=g)])
    ids = torch.cat([ids, torch.full((max(0, n - ids.numel()),), 4999, device="cuda")])[:n]
    ids = ids[torch.randperm(n, device="cuda", generator=g)]
    _check(ids, _rows(n, d, dtype), V, scale=2.0, dtype=dtype)
    # the first token is padding, a part of the ids lies outside the table: they are sorted behind all others, into later blocks of a run
    ids[::17] = 70000
    ids[5::170] = -3
    _check(ids, _rows(n, d, dtype), V, padding=0, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [128 * 96, 128 * 96 + 1, 128 * 96 - 1])
def test_tokens_that_fill_blocks_and_runs(n):
    """Each token 32 positions, then 64, 128, 256: every one begins and ends at a block's border, the larger ones at runs' borders."""
    d = 128 * 64 * 148 * 2 * 128 // (128 * 96) + 128               # runs of 128
    assert _run_length(n, d) == 128
    for size in (32, 64, 128, 256):
        ids = torch.arange(n, device="cuda") // size
        g = torch.Generator(device="cuda").manual_seed(size)
        _check(ids[torch.randperm(n, device="cuda", generator=g)], _rows(n, d, torch.bfloat16), n // 32 + 2, dtype=torch.bfloat16)
    # all but the first 5 positions of the last run have no gradient
    ids = torch.arange(n, device="cuda") // 64
    ids[128 * 95 + 5:] = -1
    _check(ids, _rows(n, d, torch.bfloat16), n // 32 + 2, dtype=torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,d", [(40000, 300000, 24), (3000, 300000, 40), (40000, 50304, 64), (70001, 131071, 16), (33000, 262144, 8), (33000, 262143, 8)])
def test_passes_and_digits_of_the_sort(n, V, d):
    """Tables of up to 18 and more bits (three passes), n above and below 32,768 (CTAs of 1,024 and of 256)."""
    g = torch.Generator(device="cuda").manual_seed(V)
    ids = torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, torch.randint(0, V, (n,), device="cuda", generator=g),
                      V - 1 - torch.randint(0, 40, (n,), device="cuda", generator=g))
    _check(ids, _rows(n, d), V, padding=V - 1)
    _check(ids.int(), _rows(n, d), V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.float16, 2 * 2**20 + 1), (torch.bfloat16, 2**22 + 1), (torch.float32, 2**21 + 37)])
def test_rows_of_any_width_that_is_accepted(dtype, d):
    """Odd widths are read an element at a time, 32 columns a warp: more than 65,535 slabs."""
    from machinelearning_b200 import token_embedding
    w = torch.zeros(3, d, device="cuda", dtype=dtype)
    ids = torch.tensor([1, 2] * 17, device="cuda")
    assert token_embedding.supports(ids, w)
    _check(ids, _rows(34, d, dtype), 3, dtype=dtype)
