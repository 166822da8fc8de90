"""The head of a language model with its cross entropy, without the logits.

``linear_cross_entropy(x, weight, targets)`` is ``F.cross_entropy(x @ weight.T, targets)`` -- nanolab's ``lm_head`` and loss
(``nanolab/model.py:364-453``) -- with gradients of ``x`` and ``weight``.  The logits of 65,536 tokens over 50,304 words are
13 GB in float32; here a tile of them lives in tensor memory until its maximum and sum of exponentials are known, and the
backward forms them again, a piece of the vocabulary at a time (``csrc/loss.cu``, ``csrc/loss_tc.cu``).

An ``autograd`` node over the C entry points.  No CPU path: ``supports`` says whether a call can run; the function
raises otherwise.
"""
from __future__ import annotations

import torch

from . import _lib, flash_cuda
from .value_gate import _DTYPE_CODE, _lib_or_raise, _stream

REDUCTIONS = {"none": _lib.REDUCE_NONE, "mean": _lib.REDUCE_MEAN, "sum": _lib.REDUCE_SUM}
MAX_EXTENT = 1 << 30                              # rows, words
MAX_WIDTH = 1 << 24


def compute_dtype(x: torch.Tensor, weight: torch.Tensor) -> torch.dtype | None:
    """What the products run in: the autocast dtype under CUDA autocast, else the common dtype (``None``: there is none)."""
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda")
    return x.dtype if x.dtype == weight.dtype else None


def supports(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor) -> bool:
    """``x [..., d]``, ``weight [V, d]``, ``targets [...]`` of int32 or int64, on one CUDA device; float32, float16 or
    bfloat16, of one dtype unless autocast says which."""
    return (x.is_cuda and weight.device == x.device and targets.device == x.device and x.dim() >= 1 and weight.dim() == 2
            and x.dtype in _DTYPE_CODE and weight.dtype in _DTYPE_CODE and compute_dtype(x, weight) in _DTYPE_CODE
            and x.shape[-1] == weight.shape[1] and 1 <= weight.shape[1] <= MAX_WIDTH and 1 <= weight.shape[0] <= MAX_EXTENT
            and targets.dtype in (torch.int32, torch.int64) and targets.shape == x.shape[:-1] and targets.numel() <= MAX_EXTENT)


def fwd(x, weight, targets, ignore_index: int, reduction: str, dtype: torch.dtype):
    """(loss float32, tape) through the C ABI: contiguous tensors."""
    lib = _lib_or_raise()
    if x.device.index not in flash_cuda._status_words:
        flash_cuda._watch_device(lib, x.device.index)
    n, (V, d) = targets.numel(), weight.shape
    xc, wc, dc = _DTYPE_CODE[x.dtype], _DTYPE_CODE[weight.dtype], _DTYPE_CODE[dtype]
    loss = torch.empty(targets.shape if reduction == "none" else (), dtype=torch.float32, device=x.device)
    with flash_cuda._on_device(x.device.index):
        tape = torch.empty(lib.nlfa_linear_ce_tape_bytes(weight.data_ptr(), n, V, d, xc, wc, dc), dtype=torch.uint8,
                           device=x.device)
        scratch = torch.empty(lib.nlfa_linear_ce_scratch_bytes(n, V, d, xc, wc, dc, 0), dtype=torch.uint8, device=x.device)
        st = lib.nlfa_linear_ce_fwd(x.data_ptr(), xc, weight.data_ptr(), wc, dc, targets.data_ptr(), targets.element_size(),
                                    n, V, d, ignore_index, REDUCTIONS[reduction], loss.data_ptr(), tape.data_ptr(),
                                    tape.numel(), scratch.data_ptr(), scratch.numel(), _stream(x))
    _lib.check("nlfa_linear_ce_fwd", st)
    return loss, tape


def bwd(grad, x_shape, x_dtype, weight, targets, tape, ignore_index: int, reduction: str, dtype: torch.dtype,
        want_dx: bool = True, want_dw: bool = True):
    """(dx, dw), ``None`` where not wanted; ``grad`` float32."""
    lib = _lib_or_raise()
    dx = torch.empty(x_shape, dtype=x_dtype, device=weight.device) if want_dx else None
    dw = torch.empty_like(weight) if want_dw else None
    n, V, d = targets.numel(), weight.shape[0], weight.shape[1]
    xc, wc, dc = _DTYPE_CODE[x_dtype], _DTYPE_CODE[weight.dtype], _DTYPE_CODE[dtype]
    with flash_cuda._on_device(weight.device.index):
        scratch = torch.empty(lib.nlfa_linear_ce_scratch_bytes(n, V, d, xc, wc, dc, 1), dtype=torch.uint8, device=weight.device)
        st = lib.nlfa_linear_ce_bwd(grad.data_ptr(), weight.data_ptr(), wc, xc, dc, targets.data_ptr(), targets.element_size(),
                                    n, V, d, ignore_index, REDUCTIONS[reduction], tape.data_ptr(), tape.numel(),
                                    dx.data_ptr() if want_dx else None, dw.data_ptr() if want_dw else None,
                                    scratch.data_ptr(), scratch.numel(), _stream(weight))
    _lib.check("nlfa_linear_ce_bwd", st)
    return dx, dw


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction, dtype):
        loss, tape = fwd(x, weight, targets, ignore_index, reduction, dtype)
        ctx.save_for_backward(weight, targets, tape)
        ctx.meta = (x.shape, x.dtype, ignore_index, reduction, dtype)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, targets, tape = ctx.saved_tensors
        x_shape, x_dtype, ignore_index, reduction, dtype = ctx.meta
        dx, dw = bwd(grad.to(torch.float32).contiguous(), x_shape, x_dtype, weight, targets, tape, ignore_index, reduction,
                     dtype, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dw, None, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -1,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of ``x @ weight.T`` (``x [..., d]``, ``weight [V, d]``) against ``targets [...]``.

    ``reduction``: ``"mean"`` over the targets that are not ``ignore_index`` (nanolab's -1; NaN when there is none),
    ``"sum"``, or ``"none"`` (the shape of ``targets``, zero where ignored).  The loss is float32; gradients have the
    dtypes of ``x`` and ``weight``.  Under CUDA autocast the products run in the autocast dtype, whatever the tensors'.
    A target outside the vocabulary gives a NaN loss and NaN gradients; rows that are ignored reach nothing, whatever ``x`` holds there.
    Where the products run in float32, infinities (and values above bf16's largest, 3.39e38) make every logit they enter NaN, also the -inf
    that masks a word: a word is masked in 16 bits, or left out of ``weight``.
    """
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(REDUCTIONS)}, got {reduction!r}")
    if flash_cuda._load() is not None and not torch.compiler.is_compiling():
        loss = flash_cuda._host.linear_ce(x, weight, targets, ignore_index, REDUCTIONS[reduction])
        if loss is not None:
            return loss
    if not supports(x, weight, targets):
        raise ValueError(f"linear_cross_entropy: unsupported inputs (x={tuple(x.shape)}/{x.dtype} on {x.device}, "
                         f"weight={tuple(weight.shape)}/{weight.dtype}, targets={tuple(targets.shape)}/{targets.dtype})")
    dtype = compute_dtype(x, weight)
    if torch.compiler.is_compiling():
        from . import compile_ops              # registered operators: one graph node instead of a graph break
        return compile_ops.linear_cross_entropy(x, weight, targets, int(ignore_index), reduction, dtype)
    x, weight, targets = x.contiguous(), weight.contiguous(), targets.contiguous()
    if not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):
        return fwd(x, weight, targets, int(ignore_index), reduction, dtype)[0]
    return _LinearCrossEntropyFn.apply(x, weight, targets, int(ignore_index), reduction, dtype)
