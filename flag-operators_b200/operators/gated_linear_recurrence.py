"""gated_linear_recurrence — a per-channel gated recurrence over a long axis, and its gradients.

    gated_linear_recurrence(x, g, beta, decay=None, *, decay_scale=1.0, initial_state=None,
                            reset=None, output_final_state=False) -> h  (or (h, h_T))
    gated_linear_recurrence_step(x, g, beta, state, decay=None, *, decay_scale=1.0) -> h

    h_t = a_t h_{t-1} + b_t , per channel

Without `decay` the gates are values, as in chunk_gated_delta_rule: a_t = g_t,
b_t = beta_t x_t.  With `decay` ([C]) they are logits, and the input is scaled so
that the state keeps its variance:
    a_t = exp(-decay_scale softplus(decay) sigmoid(g_t))
    b_t = sqrt(1 - a_t^2) sigmoid(beta_t) x_t      (decay_scale finite, not negative)

x: [B, L, C] fp32 / fp16 / bf16; g, beta: [B, L, C] of x's dtype or both fp32 (gates that are
values near 1 need fp32: bf16 has no number between 0.996 and 1).  x, g and beta may be
views whose last dimension is contiguous, such as column blocks of one projection; anything
else is copied.  h has x's dtype; states are fp32 [B, C].
  initial_state   the state before the first token (zeros if None)
  reset           bool [B, L]: steps that start again from nothing (a_t = 0), for packed sequences;
                  nothing in front of such a step reaches it, NaN and infinite gates included
  output_final_state   also return the state after the last token

Gates above 1 make the state grow; their product over any 128 consecutive steps has to stay
within the fp32 range (over an empty state it may leave it).
A padded step that keeps the state (g = 1, beta = 0 as values; g = -inf as logits) must hold
a finite x.  The state is fp32 throughout and h is rounded once.

All of x, g, beta, decay and initial_state are differentiable, once, in reverse mode (csrc/gated_recurrence.cu;
the backward reads x, g, beta and dh and recomputes the states from fp32 checkpoints every
64 steps).  gated_linear_recurrence_step is for decoding: x, g, beta [B, C], `state` [B, C] fp32
is overwritten (it must not share memory with the other arguments), and nothing is differentiated.
With `reset`, a NaN or infinity in the state in front of a run of gates whose product is 0 may not
reach the steps behind it.
"""
from __future__ import annotations

import ctypes
import logging
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

logger = logging.getLogger(__name__)

CHECKPOINT = 64  # FO_GLR_CHECKPOINT of include/flagops.h


def _check_gates(op, x, g, beta, decay, scale):
    if g.shape != x.shape or beta.shape != x.shape:
        raise ValueError(f"{op}: g shape {tuple(g.shape)} and beta shape {tuple(beta.shape)} must be "
                         f"x's {tuple(x.shape)}")
    if g.dtype != beta.dtype or g.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{op}: g ({g.dtype}) and beta ({beta.dtype}) must both have x's dtype "
                        f"({x.dtype}) or both be float32")
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"{op}: dtype {x.dtype} is not supported")
    if decay is not None and decay.shape != x.shape[-1:]:
        raise ValueError(f"{op}: decay shape {tuple(decay.shape)}, expected ({x.shape[-1]},)")
    if not (math.isfinite(scale) and scale >= 0):  # a gate above 1 has no root of 1 - a^2
        raise ValueError(f"{op}: decay_scale must be finite and not negative, got {scale}")
    dev = x.device
    if g.device != dev or beta.device != dev or (decay is not None and decay.device != dev):
        raise ValueError(f"{op}: g, beta and decay must be on the same device as x")


def _rows(t):
    """t itself where its last dimension is contiguous, else a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


_Three, _Six = ctypes.c_int64 * 3, ctypes.c_int64 * 6


def _strides(x, g, beta):
    if x.dim() == 2:
        return _Three(x.stride(0), g.stride(0), beta.stride(0))
    return _Six(x.stride(0), x.stride(1), g.stride(0), g.stride(1), beta.stride(0), beta.stride(1))


def _forward(x, g, beta, decay, h0, reset, scale, want_state, want_ckpt):
    B, L, C = x.shape
    h = x.new_empty((B, L, C))
    hT = torch.empty((B, C), dtype=torch.float32, device=x.device) if want_state else None
    ckpt = torch.empty((B, -(-L // CHECKPOINT), C), dtype=torch.float32, device=x.device) \
        if want_ckpt else None
    with _lib.on_device(x):
        _lib.call("fo_glr_fwd", _lib.ptr(x), _lib.ptr(g), _lib.ptr(beta), _lib.ptr(decay),
                  _lib.ptr(h0), _lib.ptr(reset), _lib.ptr(h), _lib.ptr(hT), _lib.ptr(ckpt), B, L, C,
                  _strides(x, g, beta), scale, _lib.dtype_code(x.dtype), _lib.dtype_code(g.dtype),
                  _lib.stream_of(x))
    return h, hT, ckpt


def _backward(x, g, beta, decay, reset, ckpt, scale, dh, dhT, need_dh0, need_ddecay):
    B, L, C = x.shape
    dev = x.device
    dh = torch.zeros((B, L, C), dtype=x.dtype, device=dev) if dh is None \
        else dh.to(x.dtype).contiguous()
    if dhT is not None:
        dhT = dhT.to(torch.float32).contiguous()
    dx, dg, dbeta = x.new_empty((B, L, C)), g.new_empty((B, L, C)), g.new_empty((B, L, C))
    dh0 = torch.empty((B, C), dtype=torch.float32, device=dev) if need_dh0 else None
    ddecay = torch.empty(C, dtype=torch.float32, device=dev) if need_ddecay else None
    ws, nbytes = None, ctypes.c_int64(0)
    with _lib.on_device(x):
        if need_ddecay:
            _lib.call("fo_glr_bwd_workspace_bytes", B, L, C, ctypes.byref(nbytes))
            ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
        _lib.call("fo_glr_bwd", _lib.ptr(x), _lib.ptr(g), _lib.ptr(beta), _lib.ptr(decay),
                  _lib.ptr(reset), _lib.ptr(ckpt), _lib.ptr(dh), _lib.ptr(dhT), _lib.ptr(dx),
                  _lib.ptr(dg), _lib.ptr(dbeta), _lib.ptr(dh0), _lib.ptr(ddecay), B, L, C,
                  _strides(x, g, beta), scale, _lib.dtype_code(x.dtype), _lib.dtype_code(g.dtype),
                  _lib.ptr(ws), nbytes.value, _lib.stream_of(x))
    return dx, dg, dbeta, dh0, ddecay


class _GatedLinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, beta, decay, h0, reset, scale, want_state):
        h, hT, ckpt = _forward(x, g, beta, decay, h0, reset, scale, want_state, True)
        ctx.save_for_backward(x, g, beta, decay, reset, ckpt)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (h, hT) if want_state else h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dhT=None):
        x, g, beta, decay, reset, ckpt = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dh is None and dhT is None:
            return (None,) * 8
        dx, dg, dbeta, dh0, ddecay = _backward(x, g, beta, decay, reset, ckpt, ctx.scale, dh, dhT,
                                               need[4], need[3])
        return (dx if need[0] else None, dg if need[1] else None, dbeta if need[2] else None,
                ddecay, dh0, None, None, None)


def gated_linear_recurrence(
    x: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    decay: torch.Tensor | None = None,
    *,
    decay_scale: float = 1.0,
    initial_state: torch.Tensor | None = None,
    reset: torch.Tensor | None = None,
    output_final_state: bool = False,
):
    """h (or (h, h_T)) of the recurrence over dim 1; see the module's documentation."""
    logger.debug("FLAG-OPS GATED_LINEAR_RECURRENCE")
    op = "gated_linear_recurrence"
    _lib.require_cuda(x, op)
    _lib.refuse_tangents(op, x, g, beta, decay, initial_state)
    if x.dim() != 3:
        raise ValueError(f"{op}: x must be [B, L, C], got shape {tuple(x.shape)}")
    scale = float(decay_scale)
    _check_gates(op, x, g, beta, decay, scale)
    B, L, C = x.shape
    h0 = initial_state
    if h0 is not None:
        if h0.shape != (B, C):
            raise ValueError(f"{op}: initial_state shape {tuple(h0.shape)}, expected ({B}, {C})")
        if h0.device != x.device:
            raise ValueError(f"{op}: initial_state must be on the same device as x")
        h0 = h0.to(torch.float32).contiguous()
    if reset is not None:
        if reset.dtype != torch.bool or reset.shape != (B, L) or reset.device != x.device:
            raise ValueError(f"{op}: reset must be a bool tensor of shape ({B}, {L}) on x's device, got "
                             f"{reset.dtype} {tuple(reset.shape)} on {reset.device}")
        reset = reset.contiguous()
    if decay is not None:
        decay = decay.to(torch.float32).contiguous()
    x, g, beta = _rows(x), _rows(g), _rows(beta)
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or beta.requires_grad
                                    or (decay is not None and decay.requires_grad)
                                    or (h0 is not None and h0.requires_grad)):
        return _GatedLinearRecurrence.apply(x, g, beta, decay, h0, reset, scale,
                                            bool(output_final_state))
    h, hT, _ = _forward(x, g, beta, decay, h0, reset, scale, output_final_state, False)
    return (h, hT) if output_final_state else h


def gated_linear_recurrence_step(
    x: torch.Tensor,
    g: torch.Tensor,
    beta: torch.Tensor,
    state: torch.Tensor,
    decay: torch.Tensor | None = None,
    *,
    decay_scale: float = 1.0,
) -> torch.Tensor:
    """One token of every sequence: overwrites `state` with h_t and returns it in x's dtype."""
    op = "gated_linear_recurrence_step"
    _lib.require_cuda(x, op)
    _lib.refuse_tangents(op, x, g, beta, decay, state)
    if x.dim() != 2:
        raise ValueError(f"{op}: x must be [B, C], got shape {tuple(x.shape)}")
    scale = float(decay_scale)
    _check_gates(op, x, g, beta, decay, scale)
    if state.shape != x.shape or state.dtype != torch.float32 or state.device != x.device \
            or not state.is_contiguous():
        raise ValueError(f"{op}: state must be a contiguous float32 tensor of shape {tuple(x.shape)} on "
                         f"x's device, got {state.dtype} {tuple(state.shape)} on {state.device}")
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or beta.requires_grad
                                    or state.requires_grad
                                    or (decay is not None and decay.requires_grad)):
        raise RuntimeError(f"{op}: overwrites its state and is not differentiable; call it under "
                           f"torch.no_grad() or use gated_linear_recurrence")
    if decay is not None:
        decay = decay.to(torch.float32).contiguous()
    x, g, beta = _rows(x), _rows(g), _rows(beta)
    B, C = x.shape
    h = x.new_empty((B, C))
    with _lib.on_device(x):
        _lib.call("fo_glr_step", _lib.ptr(x), _lib.ptr(g), _lib.ptr(beta), _lib.ptr(decay),
                  _lib.ptr(state), _lib.ptr(h), B, C, _strides(x, g, beta), scale,
                  _lib.dtype_code(x.dtype), _lib.dtype_code(g.dtype), _lib.stream_of(x))
    if not state.is_inference():  # a graph that kept the old state raises instead of using the new one
        torch.autograd.graph.increment_version(state)
    return h


def timeouts() -> int:
    """Threads that gave up a wait between CTAs or warps on the current device since the library was
    loaded (0 in a healthy run; the outputs of such a call are not complete)."""
    c = ctypes.c_uint(0)
    _lib.call("fo_glr_timeouts", ctypes.byref(c))
    return int(c.value)
