"""The gated feed-forward layer: ``down(f(gate(x)) * up(x))`` and its gradients.

``gated_ffn(x, w_gate, w_up, w_down)`` is nanolab's ``SwiGLU`` (``nanolab/model.py:29-43``; ``f`` may be another one).  Where there are many tokens both projections,
the activation and the product are one kernel, the projection down another; the backward is two more.  Up to 256 tokens with gradients, 64 without, and where few tiles have long sums, the products
are formed in parts by the whole GPU and ``f`` is a kernel of its own; a few tokens without gradients have kernels of their own (``csrc/ffn.cu``, ``csrc/ffn_tc.cu``, ``csrc/ffn_few.cu``).
Kept for the backward: the hidden values and what turns their gradient into the projections', 6 bytes for each of the ``F`` hidden values of a token in
bfloat16 (float16 10, float32 14; torch's own graph of the same layer keeps 8, in float32 16).

An ``autograd`` node over the C entry points.  No CPU path: ``supports`` says whether a call can run; the function raises otherwise.
"""
from __future__ import annotations

import torch

from . import _lib, flash_cuda
from .head_loss import compute_dtype
from .value_gate import _DTYPE_CODE, _lib_or_raise, _stream

ACTIVATIONS = {"silu": _lib.FFN_SILU, "gelu": _lib.FFN_GELU, "relu": _lib.FFN_RELU}
MAX_EXTENT = 1 << 30                              # tokens
MAX_WIDTH = 1 << 24


def supports(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> bool:
    """``x [..., d]``, ``w_gate`` and ``w_up [F, d]``, ``w_down [o, F]`` on one CUDA device; float32, float16 or bfloat16, of one dtype unless
    autocast says which (the weights of one in any case)."""
    weights = (w_gate, w_up, w_down)
    return (x.is_cuda and x.dim() >= 1 and all(w.device == x.device and w.dim() == 2 and w.dtype == w_gate.dtype for w in weights)
            and x.dtype in _DTYPE_CODE and w_gate.dtype in _DTYPE_CODE and compute_dtype(x, w_gate) in _DTYPE_CODE
            and w_up.shape == w_gate.shape and w_gate.shape[1] == x.shape[-1] and w_down.shape[1] == w_gate.shape[0]
            and all(1 <= n <= MAX_WIDTH for n in (*w_gate.shape, w_down.shape[0])) and x.numel() // x.shape[-1] <= MAX_EXTENT)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _sizes(x_shape, w_gate_shape, o):
    n = 1
    for e in x_shape[:-1]:
        n *= e
    return n, w_gate_shape[1], w_gate_shape[0], o


def copies_of(x, w_gate, w_up, w_down, dtype: torch.dtype, train: bool) -> int:
    """Which of the four (bits 0 to 3) the tape gets copies of: where the products cannot read them as they lie."""
    return _lib_or_raise().nlfa_gated_ffn_copies(x.data_ptr(), _DTYPE_CODE[x.dtype], w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                                                 _DTYPE_CODE[w_gate.dtype], _DTYPE_CODE[dtype], x.numel() // x.shape[-1],
                                                 w_gate.shape[1], w_gate.shape[0], train)


def fwd(x, w_gate, w_up, w_down, activation: str, dtype: torch.dtype, train: bool):
    """(y, tape, copies) through the C ABI: contiguous tensors.  Without ``train`` the tape is workspace."""
    lib = _lib_or_raise()
    if x.device.index not in flash_cuda._status_words:
        flash_cuda._watch_device(lib, x.device.index)
    sizes = _sizes(x.shape, w_gate.shape, w_down.shape[0])
    xc, wc, dc = _DTYPE_CODE[x.dtype], _DTYPE_CODE[w_gate.dtype], _DTYPE_CODE[dtype]
    weights = (w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr())
    y = torch.empty((*x.shape[:-1], w_down.shape[0]), dtype=dtype, device=x.device)
    with flash_cuda._on_device(x.device.index):
        copies = copies_of(x, w_gate, w_up, w_down, dtype, train)
        tape = torch.empty(lib.nlfa_gated_ffn_tape_bytes(*sizes, dc, copies, train), dtype=torch.uint8, device=x.device)
        scratch = torch.empty(lib.nlfa_gated_ffn_scratch_bytes(*sizes, dc, copies, train, 0), dtype=torch.uint8, device=x.device)
        st = lib.nlfa_gated_ffn_fwd(x.data_ptr(), xc, *weights, wc, dc, ACTIVATIONS[activation], *sizes, y.data_ptr(), copies, train,
                                    tape.data_ptr(), tape.numel(), scratch.data_ptr(), scratch.numel(), _stream(x))
    _lib.check("nlfa_gated_ffn_fwd", st)
    return y, tape, copies


def bwd(dy, x, w_gate, w_up, w_down, tape, copies: int, shapes, x_dtype, w_dtype, activation: str, want=(True, True, True, True)):
    """(dx, dw_gate, dw_up, dw_down), ``None`` where not wanted; ``dy`` contiguous, in the products' dtype.  Inputs that the tape has copies of may
    be ``None``; ``shapes``: of the four."""
    lib = _lib_or_raise()
    sizes = _sizes(shapes[0], shapes[1], shapes[3][0])
    dc = _DTYPE_CODE[dy.dtype]
    out = [torch.empty(s, dtype=x_dtype if i == 0 else w_dtype, device=dy.device) if want[i] else None for i, s in enumerate(shapes)]
    with flash_cuda._on_device(dy.device.index):
        scratch = torch.empty(lib.nlfa_gated_ffn_scratch_bytes(*sizes, dc, copies, True, 1), dtype=torch.uint8, device=dy.device)
        st = lib.nlfa_gated_ffn_bwd(dy.data_ptr(), _ptr(x), _DTYPE_CODE[x_dtype], _ptr(w_gate), _ptr(w_up), _ptr(w_down), _DTYPE_CODE[w_dtype],
                                    dc, ACTIVATIONS[activation], *sizes, copies, tape.data_ptr(), tape.numel(), *(_ptr(t) for t in out),
                                    scratch.data_ptr(), scratch.numel(), _stream(dy))
    _lib.check("nlfa_gated_ffn_bwd", st)
    return out


class _GatedFfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, dtype):
        y, tape, copies = fwd(x, w_gate, w_up, w_down, activation, dtype, True)
        inputs = (x, w_gate, w_up, w_down)
        ctx.save_for_backward(tape, *(None if copies >> i & 1 else t for i, t in enumerate(inputs)))
        ctx.meta = (copies, [t.shape for t in inputs], x.dtype, w_gate.dtype, activation)
        ctx.dtype = dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        tape, *inputs = ctx.saved_tensors
        grads = bwd(dy.to(ctx.dtype).contiguous(), *inputs, tape, *ctx.meta, ctx.needs_input_grad[:4])
        return *grads, None, None


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``(f(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``: ``x [..., d]``, ``w_gate`` and ``w_up [F, d]``, ``w_down [o, F]``, the result ``[..., o]``.

    ``activation``: ``"silu"`` (nanolab's SwiGLU), ``"gelu"`` (with erf) or ``"relu"``.  The result has the inputs' dtype, or the autocast dtype under CUDA
    autocast, in which the products run then; gradients have the dtypes of ``x`` and the weights.  Sums are float32.  In float32 the products take
    finite values below 3.39e38; an infinity makes what it enters NaN.  Any number of tokens from none on; bit-reproducible.
    """
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if flash_cuda._load() is not None and not torch.compiler.is_compiling():
        y = flash_cuda._host.gated_ffn(x, w_gate, w_up, w_down, code)
        if y is not None:
            return y
        flash_cuda.refuse_tangents("gated_ffn", x, w_gate, w_up, w_down)
    if not supports(x, w_gate, w_up, w_down):
        said = ", ".join(f"{n}={tuple(t.shape)}/{t.dtype} on {t.device}"
                         for n, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)))
        raise ValueError(f"gated_ffn: unsupported inputs ({said})")
    dtype = compute_dtype(x, w_gate)
    if torch.compiler.is_compiling():
        from . import compile_ops              # registered operators: one graph node instead of a graph break
        return compile_ops.gated_ffn(x, w_gate, w_up, w_down, activation, dtype)
    inputs = [t.contiguous() for t in (x, w_gate, w_up, w_down)]
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in inputs)):
        return fwd(*inputs, activation, dtype, False)[0]
    return _GatedFfnFn.apply(*inputs, activation, dtype)
