"""residual_rms_norm — the norms, gate and residual update between two blocks, in one kernel.

    residual_rms_norm(y, residual, weight, *, post_weight=None, gate=None,
                      gate_activation="silu", scale=1.0, eps=1e-5) -> (out, new_residual)

    p = rms_norm(y) * post_weight       (y itself without post_weight)
    u = act(gate) * p                   (p itself without a gate)
    new_residual = residual + scale * u
    out = rms_norm(new_residual) * weight

y (a block's output), residual and gate are [..., N] of one dtype (fp32 / fp16 / bf16); weight,
post_weight and a tensor `scale` are [N], all of the rows' dtype or all fp32; `scale` may also be a
number.  gate_activation is "silu" or "sigmoid" ("none": no gate).  out is the next block's
input and new_residual the stream to add its output to.  The second norm takes the sum in fp32,
before it is rounded to new_residual.  Row-strided views (column blocks of a projection) are read
in place.

Differentiable, once and in reverse mode, in every tensor argument (csrc/residual_norm.cu); sums over rows are in
a fixed order.  A gate shared by several rows may be passed expanded: autograd adds its gradient up.
"""
from __future__ import annotations

import ctypes
import logging

import torch
from torch.autograd.function import once_differentiable

from . import _lib

logger = logging.getLogger(__name__)

_ACT = {"none": 0, "silu": 1, "sigmoid": 2}  # enum fo_gate_act of include/flagops.h


def _rows(t, N):
    """(t, row stride) with t readable as [M, N] rows: t itself where it is, else a copy."""
    if t.is_contiguous():
        return t, N
    ok, ld, expected = t.stride(-1) == 1 or N == 1, N, None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if expected is None:  # the innermost dimension of rows
            ld = stride
            ok = ok and ld >= N
        else:  # outer dimensions have to fold into the same row index
            ok = ok and stride == expected
        expected = stride * size
    return (t, ld) if ok else (t.contiguous(), N)


def _inv_ptrs(inv, M):
    if inv is None:
        return None, None
    p = inv.data_ptr()
    return ctypes.c_void_p(p), ctypes.c_void_p(p + 4 * M)


def _forward(y, residual, weight, post_weight, gate, act, scale, eps, keep):
    N = weight.numel()
    M = y.numel() // N
    y, y_ld = _rows(y, N)
    residual, r_ld = _rows(residual, N)
    gate, g_ld = _rows(gate, N) if gate is not None else (None, 0)
    dev = y.device
    out, res = y.new_empty(y.shape), y.new_empty(y.shape)
    inv = torch.empty(2 * M, dtype=torch.float32, device=dev) if keep else None  # inv1, inv2
    sv, s = (scale, 1.0) if isinstance(scale, torch.Tensor) else (None, scale)
    with _lib.on_device(y):
        _lib.call("fo_residual_rms_norm_fwd", _lib.ptr(y), _lib.ptr(residual), _lib.ptr(weight),
                  _lib.ptr(post_weight), _lib.ptr(gate), _lib.ptr(sv), s, _lib.ptr(out),
                  _lib.ptr(res), *_inv_ptrs(inv, M), M, N, y_ld, r_ld, g_ld, eps, act,
                  _lib.dtype_code(y.dtype), _lib.dtype_code(weight.dtype), _lib.stream_of(y))
    return out, res, inv


class _ResidualRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, post_weight, gate, scale, act, eps):
        out, res, inv = _forward(y, residual, weight, post_weight, gate, act, scale, eps, True)
        sv = scale if isinstance(scale, torch.Tensor) else None
        ctx.save_for_backward(y, residual, weight, post_weight, gate, sv, inv)
        ctx.s = 1.0 if sv is not None else scale
        ctx.act = act
        ctx.set_materialize_grads(False)
        return out, res

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dres):
        y, residual, weight, post_weight, gate, sv, inv = ctx.saved_tensors
        if dout is None and dres is None:
            return (None,) * 8
        N = weight.numel()
        M = y.numel() // N
        y, y_ld = _rows(y, N)
        residual, r_ld = _rows(residual, N)
        gate, g_ld = _rows(gate, N) if gate is not None else (None, 0)
        dev = y.device
        dout = None if dout is None else dout.to(y.dtype).contiguous()
        dres = None if dres is None else dres.to(y.dtype).contiguous()
        dy, dr = y.new_empty(y.shape), y.new_empty(y.shape)
        dgate = y.new_empty(y.shape) if gate is not None else None
        dw = torch.empty_like(weight)
        dwp = torch.empty_like(post_weight) if post_weight is not None else None
        ds = torch.empty_like(sv) if sv is not None else None
        nbytes = ctypes.c_int64(0)
        with _lib.on_device(y):
            _lib.call("fo_residual_rms_norm_bwd_workspace_bytes", M, N, ctypes.byref(nbytes))
            ws = torch.empty(max(nbytes.value, 1), dtype=torch.uint8, device=dev)
            _lib.call("fo_residual_rms_norm_bwd", _lib.ptr(dout), _lib.ptr(dres), _lib.ptr(y),
                      _lib.ptr(residual), _lib.ptr(weight), _lib.ptr(post_weight), _lib.ptr(gate),
                      _lib.ptr(sv), ctx.s, *_inv_ptrs(inv, M), _lib.ptr(dy), _lib.ptr(dr),
                      _lib.ptr(dgate), _lib.ptr(dw), _lib.ptr(dwp), _lib.ptr(ds),
                      M, N, y_ld, r_ld, g_ld, ctx.act, _lib.dtype_code(y.dtype),
                      _lib.dtype_code(weight.dtype), _lib.ptr(ws), nbytes.value, _lib.stream_of(y))
        need = ctx.needs_input_grad
        return (dy if need[0] else None, dr if need[1] else None, dw if need[2] else None,
                dwp if need[3] else None, dgate if need[4] else None, ds if need[5] else None,
                None, None)


def residual_rms_norm(
    y: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    *,
    post_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    gate_activation: str = "silu",
    scale: float | torch.Tensor = 1.0,
    eps: float = 1e-5,
):
    """(out, new_residual); see the module's documentation."""
    logger.debug("FLAG-OPS RESIDUAL_RMS_NORM")
    op = "residual_rms_norm"
    _lib.require_cuda(y, op)
    _lib.refuse_tangents(op, y, residual, weight, post_weight, gate,
                         scale if isinstance(scale, torch.Tensor) else None)
    if y.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"{op}: dtype {y.dtype} is not supported")
    if y.dim() < 1 or y.shape[-1] < 1:
        raise ValueError(f"{op}: y must be [..., N] with N > 0, got shape {tuple(y.shape)}")
    if gate_activation not in _ACT:
        raise ValueError(f"{op}: gate_activation must be one of {sorted(_ACT)}, got "
                         f"{gate_activation!r}")
    if gate is not None and gate_activation == "none":
        raise ValueError(f"{op}: gate_activation 'none' with a gate")
    N = y.shape[-1]
    for name, t in (("residual", residual), ("gate", gate)):
        if t is None:
            continue
        if t.shape != y.shape or t.device != y.device:
            raise ValueError(f"{op}: {name} must have y's shape {tuple(y.shape)} and device, got "
                             f"{tuple(t.shape)} on {t.device}")
        if t.dtype != y.dtype:
            raise TypeError(f"{op}: {name} must have y's dtype {y.dtype}, got {t.dtype}")
    vectors = [("weight", weight), ("post_weight", post_weight)]
    if isinstance(scale, torch.Tensor):
        vectors.append(("scale", scale))
    else:
        scale = float(scale)
    for name, t in vectors:
        if t is None:
            continue
        if t.shape != (N,) or t.device != y.device:
            raise ValueError(f"{op}: {name} must have shape ({N},) on y's device, got "
                             f"{tuple(t.shape)} on {t.device}")
        if t.dtype != weight.dtype or t.dtype not in (y.dtype, torch.float32):
            raise TypeError(f"{op}: weight, post_weight and scale must all have y's dtype {y.dtype} or all "
                            f"be float32, got {name} {t.dtype}")
    weight = weight.contiguous()
    if post_weight is not None:
        post_weight = post_weight.contiguous()
    if isinstance(scale, torch.Tensor):
        scale = scale.contiguous()
    act = _ACT[gate_activation] if gate is not None else 0
    if torch.is_grad_enabled() and any(
            isinstance(t, torch.Tensor) and t.requires_grad
            for t in (y, residual, weight, post_weight, gate, scale)):
        return _ResidualRmsNorm.apply(y, residual, weight, post_weight, gate, scale, act, float(eps))
    out, res, _ = _forward(y, residual, weight, post_weight, gate, act, scale, float(eps), False)
    return out, res
