"""``torch.library`` registration of the attention kernels, for ``torch.compile``.

nanolab compiles its model when ``Config.compile`` is on (``nanolab/train.py:213-214``).
``flash_cuda.flash_attn`` is an ``autograd.Function`` around ctypes calls, which the
compiler cannot trace: the graph breaks at every layer.  Registered as custom operators
with shape functions and an autograd formula, the same calls become single opaque nodes
of the traced graph, forward and backward.

    from machinelearning_b200 import compile_ops
    y = compile_ops.flash_attn(q, k, v, scale, window=0, sinks=0)      # same contract as flash_cuda.flash_attn

``flash_cuda.flash_attn`` itself takes this route while a compiler is tracing, and so do
``qk_prologue.qk_prologue``, ``value_gate.value_blend`` and ``value_gate.head_gate`` (operators
``nlfa::qk_prologue_*``, ``nlfa::value_blend_*``, ``nlfa::head_gate_*`` below).  The operators
run only the library's kernels; there is no CPU implementation, only the shape functions
tracing needs.
"""
from __future__ import annotations

import math

import torch

from . import flash_cuda


@torch.library.custom_op("nlfa::attn_fwd", mutates_args=(), device_types="cuda")
def attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, use_mma: bool, window: int,
             sinks: int, block: int) -> tuple[torch.Tensor, torch.Tensor]:
    return flash_cuda.fwd(q, k, v, scale, use_mma, window, sinks, block)


@attn_fwd.register_fake
def _(q, k, v, scale, use_mma, window, sinks, block):
    B, T, H, _ = q.shape
    return torch.empty_like(q), q.new_empty((B, H, T), dtype=torch.float32)


@torch.library.custom_op("nlfa::attn_bwd", mutates_args=(), device_types="cuda")
def attn_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
             lse: torch.Tensor, scale: float, use_mma: bool, window: int,
             sinks: int, block: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return flash_cuda.bwd(dout.contiguous(), q, k, v, o, lse, scale, use_mma, window, sinks, block=block)


@attn_bwd.register_fake
def _(dout, q, k, v, o, lse, scale, use_mma, window, sinks, block):
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)


def _setup(ctx, inputs, output):
    q, k, v, scale, use_mma, window, sinks, block = inputs
    o, lse = output
    ctx.save_for_backward(q, k, v, o, lse)
    ctx.args = (scale, use_mma, window, sinks, block)


def _backward(ctx, dout, dlse):
    q, k, v, o, lse = ctx.saved_tensors
    dq, dk, dv = attn_bwd(dout, q, k, v, o, lse, *ctx.args)
    return dq, dk, dv, None, None, None, None, None


attn_fwd.register_autograd(_backward, setup_context=_setup)


def flash_attn(q, k, v, scale=None, use_mma=None, *, window: int = 0, sinks: int = 0, block: int = 0):
    """``flash_cuda.flash_attn`` through the registered operators (same checks, same casts)."""
    q, k, v, scale, use_mma = flash_cuda.prepare(q, k, v, scale, use_mma, window, sinks, block)
    return attn_fwd(q, k, v, float(scale), bool(use_mma), int(window), int(sinks), int(block))[0]


# ---------------------------------------------------------------- q/k prologue, value blend, head gate
from typing import Optional  # noqa: E402

from . import qk_prologue as _qp  # noqa: E402
from . import value_gate as _vg  # noqa: E402


@torch.library.custom_op("nlfa::qk_prologue_fwd", mutates_args=(), device_types="cuda")
def qk_prologue_fwd(x: torch.Tensor, weight: Optional[torch.Tensor], cos: Optional[torch.Tensor],
                    sin: Optional[torch.Tensor], eps: float, out_dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    return _qp.fwd(x, weight, cos, sin, eps, out_dtype)


@qk_prologue_fwd.register_fake
def _(x, weight, cos, sin, eps, out_dtype):
    rows = x.shape[0] * x.shape[1] * x.shape[2] if weight is not None else 1
    return x.new_empty(x.shape, dtype=out_dtype), x.new_empty((rows,), dtype=torch.float32)


@torch.library.custom_op("nlfa::qk_prologue_bwd", mutates_args=(), device_types="cuda")
def qk_prologue_bwd(gy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], cos: Optional[torch.Tensor],
                    sin: Optional[torch.Tensor], rstd: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _qp.bwd(gy.contiguous(), x, weight, cos, sin, rstd)


@qk_prologue_bwd.register_fake
def _(gy, x, weight, cos, sin, rstd):
    return torch.empty_like(x), x.new_empty((x.shape[-1] if weight is not None else 1,), dtype=torch.float32)


def _qp_setup(ctx, inputs, output):
    x, weight, cos, sin, eps, out_dtype = inputs
    ctx.save_for_backward(x, weight, cos, sin, output[1])
    ctx.has_weight = weight is not None


def _qp_backward(ctx, gy, grstd):
    x, weight, cos, sin, rstd = ctx.saved_tensors
    gx, gw = qk_prologue_bwd(gy, x, weight, cos, sin, rstd)
    return gx, (gw if ctx.has_weight else None), None, None, None, None


qk_prologue_fwd.register_autograd(_qp_backward, setup_context=_qp_setup)


def qk_prologue(x, weight, cos, sin, eps, out_dtype):
    """``qk_prologue.qk_prologue`` through the registered operators (float32 weight and tables)."""
    f32 = lambda t: None if t is None else t.to(torch.float32).contiguous()
    return qk_prologue_fwd(x.contiguous(), f32(weight), f32(cos), f32(sin), float(eps), out_dtype)[0]


@torch.library.custom_op("nlfa::value_blend_fwd", mutates_args=(), device_types="cuda")
def value_blend_fwd(v: torch.Tensor, v0: torch.Tensor, lam: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    return _vg.blend_fwd(v, v0, lam, out_dtype)


@value_blend_fwd.register_fake
def _(v, v0, lam, out_dtype):
    return v.new_empty(v.shape, dtype=out_dtype)


@torch.library.custom_op("nlfa::value_blend_bwd", mutates_args=(), device_types="cuda")
def value_blend_bwd(g: torch.Tensor, v: torch.Tensor, v0: torch.Tensor,
                    lam: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _vg.blend_bwd(g.contiguous(), v, v0, lam)


@value_blend_bwd.register_fake
def _(g, v, v0, lam):
    return torch.empty_like(v), torch.empty_like(v0), lam.new_empty((1,), dtype=torch.float32)


def _vb_setup(ctx, inputs, output):
    v, v0, lam, out_dtype = inputs
    ctx.save_for_backward(v, v0, lam)


def _vb_backward(ctx, g):
    v, v0, lam = ctx.saved_tensors
    dv, dv0, dlam = value_blend_bwd(g, v, v0, lam)
    return dv, dv0, dlam, None


value_blend_fwd.register_autograd(_vb_backward, setup_context=_vb_setup)


def value_blend(v, v0, lam, out_dtype):
    lam32 = lam.to(torch.float32).reshape(1)
    return value_blend_fwd(v.contiguous(), v0.contiguous(), lam32, out_dtype)


@torch.library.custom_op("nlfa::head_gate_fwd", mutates_args=(), device_types="cuda")
def head_gate_fwd(y: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
    return _vg.gate_fwd(y, gate)


@head_gate_fwd.register_fake
def _(y, gate):
    return torch.empty_like(y)


@torch.library.custom_op("nlfa::head_gate_bwd", mutates_args=(), device_types="cuda")
def head_gate_bwd(g: torch.Tensor, y: torch.Tensor, gate: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _vg.gate_bwd(g.contiguous().to(y.dtype), y, gate)


@head_gate_bwd.register_fake
def _(g, y, gate):
    return torch.empty_like(y), torch.empty_like(gate)


def _hg_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _hg_backward(ctx, g):
    y, gate = ctx.saved_tensors
    return head_gate_bwd(g, y, gate)


head_gate_fwd.register_autograd(_hg_backward, setup_context=_hg_setup)


def head_gate(y, gate):
    return head_gate_fwd(y.contiguous(), gate.contiguous())


# ---------------------------------------------------------------- head with its loss, token embedding
from . import head_loss as _hl  # noqa: E402
from . import token_embedding as _te  # noqa: E402


@torch.library.custom_op("nlfa::linear_ce_fwd", mutates_args=(), device_types="cuda")
def linear_ce_fwd(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int, reduction: str,
                  dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    return _hl.fwd(x, weight, targets, ignore_index, reduction, dtype)


@linear_ce_fwd.register_fake
def _(x, weight, targets, ignore_index, reduction, dtype):
    tape = torch.library.get_ctx().new_dynamic_size()
    return (x.new_empty(targets.shape if reduction == "none" else (), dtype=torch.float32),
            x.new_empty((tape,), dtype=torch.uint8))


@torch.library.custom_op("nlfa::linear_ce_bwd", mutates_args=(), device_types="cuda")
def linear_ce_bwd(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, tape: torch.Tensor,
                  ignore_index: int, reduction: str, dtype: torch.dtype, want_dx: bool,
                  want_dw: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """A gradient that is not wanted costs nothing and comes back without elements."""
    dx, dw = _hl.bwd(grad.to(torch.float32).contiguous(), x.shape, x.dtype, weight, targets, tape, ignore_index, reduction, dtype,
                     want_dx, want_dw)
    return dx if want_dx else x.new_empty(0), dw if want_dw else weight.new_empty(0)


@linear_ce_bwd.register_fake
def _(grad, x, weight, targets, tape, ignore_index, reduction, dtype, want_dx, want_dw):
    return torch.empty_like(x) if want_dx else x.new_empty(0), torch.empty_like(weight) if want_dw else weight.new_empty(0)


def _ce_setup(ctx, inputs, output):
    x, weight, targets, ignore_index, reduction, dtype = inputs
    ctx.save_for_backward(x, weight, targets, output[1])
    ctx.args = (ignore_index, reduction, dtype)


def _ce_backward(ctx, grad, gtape):
    x, weight, targets, tape = ctx.saved_tensors
    want_dx, want_dw = ctx.needs_input_grad[:2]
    dx, dw = linear_ce_bwd(grad, x, weight, targets, tape, *ctx.args, want_dx, want_dw)
    return dx if want_dx else None, dw if want_dw else None, None, None, None, None


linear_ce_fwd.register_autograd(_ce_backward, setup_context=_ce_setup)


def linear_cross_entropy(x, weight, targets, ignore_index, reduction, dtype):
    """``head_loss.linear_cross_entropy`` through the registered operators."""
    return linear_ce_fwd(x.contiguous(), weight.contiguous(), targets.contiguous(), ignore_index, reduction, dtype)[0]


@torch.library.custom_op("nlfa::embedding_fwd", mutates_args=(), device_types="cuda")
def embedding_fwd(idx: torch.Tensor, weight: torch.Tensor, scale: float, padding: int) -> torch.Tensor:
    return _te.fwd(idx, weight, scale)


@embedding_fwd.register_fake
def _(idx, weight, scale, padding):
    return weight.new_empty((*idx.shape, weight.shape[1]))


@torch.library.custom_op("nlfa::embedding_bwd", mutates_args=(), device_types="cuda")
def embedding_bwd(g: torch.Tensor, idx: torch.Tensor, rows: int, scale: float, padding: int) -> torch.Tensor:
    return _te.bwd(g.contiguous(), idx, rows, scale, padding)


@embedding_bwd.register_fake
def _(g, idx, rows, scale, padding):
    return g.new_empty((rows, g.shape[-1]))


def _te_setup(ctx, inputs, output):
    idx, weight, scale, padding = inputs
    ctx.save_for_backward(idx)
    ctx.args = (weight.shape[0], scale, padding)


def _te_backward(ctx, g):
    (idx,) = ctx.saved_tensors
    return None, embedding_bwd(g, idx, *ctx.args), None, None


embedding_fwd.register_autograd(_te_backward, setup_context=_te_setup)


def embedding(idx, weight, scale, padding):
    """``token_embedding.embedding`` through the registered operators."""
    return embedding_fwd(idx.contiguous(), weight.contiguous(), scale, padding)


# ---------------------------------------------------------------- gated recurrence
from . import gated_scan as _gs  # noqa: E402


@torch.library.custom_op("nlfa::gated_scan_fwd", mutates_args=(), device_types="cuda")
def gated_scan_fwd(gate: torch.Tensor, value: torch.Tensor, state: torch.Tensor | None, reset: torch.Tensor | None,
                   lengths: torch.Tensor | None, activation: str, train: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _gs.fwd(_gs._rows(gate), _gs._rows(value), state, reset, lengths, activation, train)


@gated_scan_fwd.register_fake
def _(gate, value, state, reset, lengths, activation, train):
    tape = torch.library.get_ctx().new_dynamic_size()
    return (gate.new_empty(gate.shape), gate.new_empty((gate.shape[0], gate.shape[2]), dtype=torch.float32),
            gate.new_empty((tape,), dtype=torch.uint8))


@torch.library.custom_op("nlfa::gated_scan_bwd", mutates_args=(), device_types="cuda")
def gated_scan_bwd(dh: torch.Tensor | None, dlast: torch.Tensor | None, gate: torch.Tensor, value: torch.Tensor,
                   reset: torch.Tensor | None, lengths: torch.Tensor | None, tape: torch.Tensor, activation: str, want_gate: bool,
                   want_value: bool, want_state: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A gradient that is not wanted costs nothing and comes back without elements."""
    dh = None if dh is None else dh.to(gate.dtype).contiguous()
    dlast = None if dlast is None else dlast.to(torch.float32).contiguous()
    grads = _gs.bwd(dh, dlast, _gs._rows(gate), _gs._rows(value), reset, lengths, tape, activation, (want_gate, want_value, want_state))
    return tuple(gate.new_empty(0) if g is None else g for g in grads)


@gated_scan_bwd.register_fake
def _(dh, dlast, gate, value, reset, lengths, tape, activation, want_gate, want_value, want_state):
    return (gate.new_empty(gate.shape if want_gate else 0), gate.new_empty(gate.shape if want_value else 0),
            gate.new_empty((gate.shape[0], gate.shape[2]), dtype=torch.float32) if want_state else gate.new_empty(0))


def _gs_setup(ctx, inputs, output):
    gate, value, _, reset, lengths, activation, _ = inputs
    ctx.save_for_backward(gate, value, reset, lengths, output[2])
    ctx.activation = activation


def _gs_backward(ctx, dh, dlast, gtape):
    gate, value, reset, lengths, tape = ctx.saved_tensors
    want = [bool(w) for w in ctx.needs_input_grad[:3]]
    grads = gated_scan_bwd(dh, dlast, gate, value, reset, lengths, tape, ctx.activation, *want)
    return *(g if w else None for g, w in zip(grads, want)), None, None, None, None


gated_scan_fwd.register_autograd(_gs_backward, setup_context=_gs_setup)


def gated_scan(gate, value, state, reset, lengths, activation):
    """``gated_scan.gated_scan`` through the registered operators."""
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (gate, value, state))
    h, last, _ = gated_scan_fwd(gate, value, state, reset, lengths, activation, train)
    return h, last


# ---------------------------------------------------------------- gated feed-forward layer
from . import gated_ffn as _gf  # noqa: E402


def _aligned(inputs):
    """On 16-byte boundaries, so that which operands the tape has copies of follows from types and sizes alone."""
    return [t if t.data_ptr() % 16 == 0 else t.clone() for t in inputs]


@torch.library.custom_op("nlfa::gated_ffn_fwd", mutates_args=(), device_types="cuda")
def gated_ffn_fwd(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str, dtype: torch.dtype,
                  train: bool) -> tuple[torch.Tensor, torch.Tensor]:
    y, tape, _ = _gf.fwd(*_aligned((x, w_gate, w_up, w_down)), activation, dtype, train)
    return y, tape if train else tape.new_empty(0)


@gated_ffn_fwd.register_fake
def _(x, w_gate, w_up, w_down, activation, dtype, train):
    tape = torch.library.get_ctx().new_dynamic_size()
    return x.new_empty((*x.shape[:-1], w_down.shape[0]), dtype=dtype), x.new_empty((tape,), dtype=torch.uint8)


@torch.library.custom_op("nlfa::gated_ffn_bwd", mutates_args=(), device_types="cuda")
def gated_ffn_bwd(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, tape: torch.Tensor,
                  activation: str, dtype: torch.dtype, want: list[bool]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """A gradient that is not wanted costs nothing and comes back without elements."""
    inputs = _aligned((x, w_gate, w_up, w_down))
    grads = _gf.bwd(dy.to(dtype).contiguous(), *inputs, tape, _gf.copies_of(*inputs, dtype, True), [t.shape for t in inputs], x.dtype, w_gate.dtype,
                    activation, want)
    return tuple(t.new_empty(0) if g is None else g for t, g in zip(inputs, grads))


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, tape, activation, dtype, want):
    return tuple(t.new_empty(t.shape if w else 0) for t, w in zip((x, w_gate, w_up, w_down), want))


def _gf_setup(ctx, inputs, output):
    *tensors, activation, dtype, _ = inputs
    ctx.save_for_backward(*tensors, output[1])
    ctx.args = (activation, dtype)


def _gf_backward(ctx, dy, gtape):
    want = [bool(w) for w in ctx.needs_input_grad[:4]]
    grads = gated_ffn_bwd(dy, *ctx.saved_tensors, *ctx.args, want)
    return *(g if w else None for g, w in zip(grads, want)), None, None, None


gated_ffn_fwd.register_autograd(_gf_backward, setup_context=_gf_setup)


def gated_ffn(x, w_gate, w_up, w_down, activation, dtype):
    """``gated_ffn.gated_ffn`` through the registered operators."""
    inputs = [t.contiguous() for t in (x, w_gate, w_up, w_down)]
    train = torch.is_grad_enabled() and any(t.requires_grad for t in inputs)
    return gated_ffn_fwd(*inputs, activation, dtype, train)[0]
