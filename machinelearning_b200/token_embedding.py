"""Token embedding: rows of a table, scaled, and the table's gradient.

``embedding(idx, weight)`` is nanolab's ``tok_emb`` (``nanolab/model.py:205-245``) as a function, with an optional factor
(``sqrt(d)`` in models that scale their embeddings).  The gradient adds each token's rows in the order of their
positions (``csrc/embedding.cu``), so it is bit-reproducible, unlike an atomic scatter.

An ``autograd`` node over the C entry points.  No CPU path: ``supports`` says whether a call can run; the function raises
otherwise.
"""
from __future__ import annotations

import torch

from . import _lib, flash_cuda
from .value_gate import _DTYPE_CODE, _lib_or_raise, _stream

MAX_EXTENT = 1 << 30                              # tokens, words
MAX_WIDTH = 1 << 24


def supports(idx: torch.Tensor, weight: torch.Tensor) -> bool:
    """``idx`` of any shape, int32 or int64, ``weight [V, d]`` float32, float16 or bfloat16, on one CUDA device."""
    return (weight.is_cuda and idx.device == weight.device and weight.dim() == 2 and weight.dtype in _DTYPE_CODE
            and idx.dtype in (torch.int32, torch.int64) and 1 <= weight.shape[0] <= MAX_EXTENT
            and 1 <= weight.shape[1] <= MAX_WIDTH and idx.numel() <= MAX_EXTENT)


def fwd(idx, weight, scale: float):
    """The rows through the C ABI: contiguous tensors."""
    lib = _lib_or_raise()
    V, d = weight.shape
    out = torch.empty((*idx.shape, d), dtype=weight.dtype, device=weight.device)
    with flash_cuda._on_device(weight.device.index):
        st = lib.nlfa_embedding_fwd(idx.data_ptr(), idx.element_size(), weight.data_ptr(), _DTYPE_CODE[weight.dtype],
                                    out.data_ptr(), idx.numel(), V, d, scale, _stream(weight))
    _lib.check("nlfa_embedding_fwd", st)
    return out


def bwd(g, idx, V: int, scale: float, padding: int):
    """dweight [V, d] of ``g [..., d]``'s dtype; ``padding`` negative: none."""
    lib = _lib_or_raise()
    d = g.shape[-1]
    dw = torch.empty((V, d), dtype=g.dtype, device=g.device)
    with flash_cuda._on_device(g.device.index):
        scratch = torch.empty(lib.nlfa_embedding_scratch_bytes(idx.numel(), V, d), dtype=torch.uint8, device=g.device)
        st = lib.nlfa_embedding_bwd(g.data_ptr(), _DTYPE_CODE[g.dtype], idx.data_ptr(), idx.element_size(), dw.data_ptr(),
                                    idx.numel(), V, d, scale, padding, scratch.data_ptr(), scratch.numel(), _stream(g))
    _lib.check("nlfa_embedding_bwd", st)
    return dw


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, idx, weight, scale, padding):
        ctx.save_for_backward(idx)
        ctx.meta = (weight.shape[0], weight.dtype, scale, padding)
        return fwd(idx, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (idx,) = ctx.saved_tensors
        V, dtype, scale, padding = ctx.meta
        return None, bwd(g.to(dtype).contiguous(), idx, V, scale, padding), None, None


def embedding(idx: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[idx]``, ``[..., d]`` in ``weight``'s dtype.

    ``padding_idx`` (negative counts from the end, as in ``nn.Embedding``): its row gets no gradient.  An id outside the
    table gives a row of NaN and no gradient (torch stops the process for one); the check would cost a synchronisation.
    """
    padding = -1
    if padding_idx is not None:
        V = weight.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {V}")
        padding = int(padding_idx) % V
    if flash_cuda._load() is not None and not torch.compiler.is_compiling():
        out = flash_cuda._host.embedding(idx, weight, scale, padding)
        if out is not None:
            return out
    if not supports(idx, weight):
        raise ValueError(f"embedding: unsupported inputs (idx={tuple(idx.shape)}/{idx.dtype} on {idx.device}, "
                         f"weight={tuple(weight.shape)}/{weight.dtype} on {weight.device})")
    if torch.compiler.is_compiling():
        from . import compile_ops              # registered operators: one graph node instead of a graph break
        return compile_ops.embedding(idx, weight, float(scale), padding)
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return fwd(idx.contiguous(), weight.contiguous(), float(scale))
    return _EmbeddingFn.apply(idx.contiguous(), weight.contiguous(), float(scale), padding)
