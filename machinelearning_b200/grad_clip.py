"""The norm of all gradients, and their clip: ``torch.nn.utils.clip_grad_norm_`` in two launches.

nanolab clips after every backward (``train.py:336-344``).  torch takes a norm per tensor, stacks them, takes their norm and multiplies
every gradient, also by one; here one pass reads all gradients, and a second one changes them only where the norm is above
the limit (``csrc/grad_clip.cu``).  Nothing synchronises, and the sums are in float64 and in a fixed order.

No CPU path: other gradients than plain float32, float16 or bfloat16 ones on one CUDA device raise ``ValueError``.
"""
from __future__ import annotations

import math

import torch

from . import _lib, flash_cuda

NORMS = {2.0: 2, math.inf: 0}
MAX_TENSORS = 64000


def supports(grads) -> bool:
    """Whether the kernels take these gradients (a list): plain tensors of their types, on one CUDA device."""
    return (0 < len(grads) <= MAX_TENSORS
            and all(g.is_cuda and g.layout == torch.strided and g.dtype in flash_cuda.SUPPORTED_DTYPES
                    and g.device == grads[0].device for g in grads))


def _norm_code(norm_type) -> int:
    code = NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return code


def _run(tensors, out, max_norm, code, scale, of_parameters):
    if flash_cuda._load() is None:
        grads = [t.grad for t in tensors if t.grad is not None] if of_parameters else tensors
        if not grads:
            return None
        if not supports(grads):
            raise ValueError("gradients must be plain float32, float16 or bfloat16 tensors on one CUDA device")
        raise RuntimeError(f"flash_cuda is unavailable ({flash_cuda.unavailable_reason()})")
    return flash_cuda._host.clip_grads(tensors, out, max_norm, code, scale, of_parameters)


def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all tensors' elements as one vector: a float32 scalar on their device (0 for no tensors)."""
    code = _norm_code(norm_type)
    grads = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not grads:
        return torch.tensor(0.0)
    return _run(grads, None, 0.0, code, False, False)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, *,
                    out=None) -> torch.Tensor:
    """Scale the gradients of ``parameters`` by ``min(1, max_norm / (norm + 1e-6))``; returns the norm before.

    As ``torch.nn.utils.clip_grad_norm_`` (norms 2 and inf).  Gradients within the limit are left untouched.  With ``out``, one dense
    tensor for each gradient there is, the clipped gradients go there -- in the type of ``out``, so 16-bit gradients can become the
    optimiser's float32 ones in the same pass -- and the gradients stay as they are.  Tensors that share memory raise
    ``ValueError``.  ``error_if_nonfinite`` waits for the norm.
    """
    code = _norm_code(norm_type)
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    out = None if out is None else list(out)
    if error_if_nonfinite:
        norm = _run(parameters, None, 0.0, code, False, True)
        if norm is not None and not math.isfinite(norm.item()):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, "
                               "so it cannot be clipped. To disable this error and scale the gradients by the non-finite "
                               "norm anyway, set `error_if_nonfinite=False`")
    norm = _run(parameters, out, float(max_norm), code, True, True)
    if norm is None:                                  # no gradients
        if out:
            raise ValueError(f"out: {len(out)} tensors for 0 gradients")
        return torch.tensor(0.0)
    return norm
