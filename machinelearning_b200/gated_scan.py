"""The gated linear recurrence of a MinGRU mixer (``nanolab/mixers.py``), over whole sequences and step by step.

``gated_scan(gate, value, state)`` walks ``h_t = (1 - s_t) h_{t-1} + s_t f(value_t)``, ``s = sigmoid(gate)``, for every channel: in one pass
over the data (``csrc/scan.cu``), where torch would join runs of 1, 2, 4, ... steps in some 2 log2(T) passes, and with gradients that
need no more than the states at every 16th step (float32: every 8th).

An ``autograd`` node over the C entry points.  No CPU path: ``supports`` says whether a call can run; the function raises otherwise.
"""
from __future__ import annotations

import torch

from . import _lib, flash_cuda
from .value_gate import _DTYPE_CODE, _lib_or_raise, _stream

ACTIVATIONS = {"none": _lib.SCAN_NONE, "positive": _lib.SCAN_POSITIVE}
MAX_EXTENT = 1 << 30                              # sequences, steps, channels


def supports(gate: torch.Tensor, value: torch.Tensor, state: torch.Tensor | None = None, reset: torch.Tensor | None = None,
             lengths: torch.Tensor | None = None) -> bool:
    """``gate`` and ``value [B, T, D]`` of one dtype (float32, float16 or bfloat16), ``state [B, D]`` of any of these, ``reset [B, T]`` bool,
    ``lengths [B]`` int32 or int64, on one CUDA device."""
    return (gate.is_cuda and value.device == gate.device and gate.dim() == 3 and value.shape == gate.shape and gate.dtype in _DTYPE_CODE
            and value.dtype == gate.dtype and all(n <= MAX_EXTENT for n in gate.shape)
            and (state is None or (state.device == gate.device and state.dtype in _DTYPE_CODE
                                   and state.shape == (gate.shape[0], gate.shape[2])))
            and (reset is None or (reset.device == gate.device and reset.dtype == torch.bool and reset.shape == gate.shape[:2]))
            and (lengths is None or (lengths.device == gate.device and lengths.dtype in (torch.int32, torch.int64)
                                     and lengths.shape == gate.shape[:1])))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _mask_args(reset, lengths):
    return _ptr(reset), _ptr(lengths), 0 if lengths is None else lengths.element_size()


def _rows(t):
    """Channels side by side; sequences and steps may have strides of their own."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _scratch(lib, gate):
    return torch.empty(lib.nlfa_gated_scan_scratch_bytes(*gate.shape, _DTYPE_CODE[gate.dtype]), dtype=torch.uint8, device=gate.device)


def fwd(gate, value, state, reset, lengths, activation: str, train: bool):
    """(h, last float32, tape) through the C ABI; no elements in ``tape`` unless ``train``."""
    lib = _lib_or_raise()
    if gate.device.index not in flash_cuda._status_words:
        flash_cuda._watch_device(lib, gate.device.index)
    B, T, D = gate.shape
    h = torch.empty((B, T, D), dtype=gate.dtype, device=gate.device)
    last = torch.empty((B, D), dtype=torch.float32, device=gate.device)
    tape = torch.empty(lib.nlfa_gated_scan_tape_bytes(B, T, D, _DTYPE_CODE[gate.dtype]) if train else 0, dtype=torch.uint8, device=gate.device)
    with flash_cuda._on_device(gate.device.index):
        scratch = _scratch(lib, gate)
        st = lib.nlfa_gated_scan_fwd(gate.data_ptr(), gate.stride(0), gate.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
                                     _DTYPE_CODE[gate.dtype], _ptr(state), *_mask_args(reset, lengths), ACTIVATIONS[activation], B, T, D,
                                     h.data_ptr(), last.data_ptr(), tape.data_ptr() if train else None, tape.numel(), scratch.data_ptr(),
                                     scratch.numel(), _stream(gate))
    _lib.check("nlfa_gated_scan_fwd", st)
    return h, last, tape


def bwd(dh, dlast, gate, value, reset, lengths, tape, activation: str, want=(True, True, True)):
    """(dgate, dvalue, dstate float32), ``None`` where not wanted; ``dh`` or ``dlast`` may be ``None`` (zeros)."""
    lib = _lib_or_raise()
    B, T, D = gate.shape
    dgate, dvalue = (torch.empty((B, T, D), dtype=gate.dtype, device=gate.device) if w else None for w in want[:2])
    dstate = torch.empty((B, D), dtype=torch.float32, device=gate.device) if want[2] else None
    with flash_cuda._on_device(gate.device.index):
        scratch = _scratch(lib, gate)
        st = lib.nlfa_gated_scan_bwd(_ptr(dh), _ptr(dlast), gate.data_ptr(), gate.stride(0), gate.stride(1), value.data_ptr(), value.stride(0),
                                     value.stride(1), _DTYPE_CODE[gate.dtype], *_mask_args(reset, lengths), ACTIVATIONS[activation], B, T, D,
                                     tape.data_ptr(), tape.numel(), _ptr(dgate), _ptr(dvalue), _ptr(dstate), scratch.data_ptr(),
                                     scratch.numel(), _stream(gate))
    _lib.check("nlfa_gated_scan_bwd", st)
    return dgate, dvalue, dstate


class _GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, value, state, reset, lengths, activation):
        h, last, tape = fwd(gate, value, state, reset, lengths, activation, True)
        ctx.save_for_backward(gate, value, reset, lengths, tape)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        gate, value, reset, lengths, tape = ctx.saved_tensors
        if dh is None and dlast is None:
            return (None,) * 6
        dh = None if dh is None else dh.to(gate.dtype).contiguous()
        dlast = None if dlast is None else dlast.to(torch.float32).contiguous()
        return *bwd(dh, dlast, gate, value, reset, lengths, tape, ctx.activation, ctx.needs_input_grad[:3]), None, None, None


def gated_scan(gate: torch.Tensor, value: torch.Tensor, state: torch.Tensor | None = None, *, activation: str = "none",
               reset: torch.Tensor | None = None, lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(h, last)``: ``h_t = (1 - sigmoid(gate_t)) h_{t-1} + sigmoid(gate_t) f(value_t)``, ``h [B, T, D]`` in the dtype of ``gate``, and the
    state behind the last step, ``[B, D]`` float32 -- the ``state`` of the next call.

    ``gate`` and ``value [B, T, D]`` may be halves of one projection's output.  ``state [B, D]`` (zeros when ``None``) is ``h_0``.
    ``activation``: ``"none"``, or ``"positive"``, MinGRU's map of its candidates: ``v + 1/2`` from zero on, ``sigmoid(v)`` below.
    ``reset [B, T]``: where true, the step begins anew (``h_{t-1}`` counts as zero): packed sequences.  ``lengths [B]``: steps from there on are padding:
    they leave the state as it is, their ``h`` is zero, and what ``gate`` and ``value`` hold there reaches nothing.
    ``T == 1`` is one decoding step.  Gradients of ``gate``, ``value`` and ``state``; bit-reproducible.
    """
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if flash_cuda._load() is not None and not torch.compiler.is_compiling():
        out = flash_cuda._host.gated_scan(gate, value, state, reset, lengths, code)
        if out is not None:
            return out
        flash_cuda.refuse_tangents("gated_scan", gate, value, state)
    if not supports(gate, value, state, reset, lengths):
        def said(t):
            return None if t is None else f"{tuple(t.shape)}/{t.dtype} on {t.device}"
        raise ValueError(f"gated_scan: unsupported inputs (gate={said(gate)}, value={said(value)}, state={said(state)}, reset={said(reset)}, "
                         f"lengths={said(lengths)})")
    state = None if state is None else state.to(torch.float32).contiguous()
    reset, lengths = (None if t is None else t.contiguous() for t in (reset, lengths))
    if torch.compiler.is_compiling():
        from . import compile_ops              # registered operators: one graph node instead of a graph break
        return compile_ops.gated_scan(gate, value, state, reset, lengths, activation)
    gate, value = _rows(gate), _rows(value)
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (gate, value, state))):
        return fwd(gate, value, state, reset, lengths, activation, False)[:2]
    return _GatedScanFn.apply(gate, value, state, reset, lengths, activation)
