"""RMS norms on both sides of a transformer block, fused with what stands next to them: the branch's gate, the residual sum
and its scale, and the 8-bit rows that `linear_int8` takes.  One launch forward (`b200moe_block_norm`), two backward
(`b200moe_block_norm_bwd`; one where no parameter takes a gradient).  The reference has no counterpart: its MoE operator starts
behind the norm and ends before the residual sum.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import MAX_ROW, ROW_TYPES, on_device, rows_of, stream_of


def _p(t):
    return None if t is None else t.data_ptr()


def _f32_bits(weight, gate, next_weight):
    f = torch.float32
    return ((weight is not None and weight.dtype == f) | (gate is not None and gate.dtype == f) << 1 |
            (next_weight is not None and next_weight.dtype == f) << 2)


def _gate_of(gate, kind):
    """(tensor, elements between its rows) as the kernels read it."""
    if gate is None:
        return None, 0
    if kind == _lib.GATE_FULL:
        return rows_of(gate)
    gate = gate.contiguous()
    return gate, 1


def _forward(y, residual, weight, gate, kind, next_weight, alpha, eps, want_h, quant, save):
    dev, H = y.device, y.shape[-1]
    y2, ys = rows_of(y)
    T = y2.shape[0]
    r2, rs = (None, 0) if residual is None else rows_of(residual)
    g2, gs = _gate_of(gate, kind)
    w = None if weight is None else weight.contiguous()
    wn = None if next_weight is None else next_weight.contiguous()
    h = torch.empty(y.shape, dtype=y.dtype, device=dev) if want_h else None
    n = q = scale = None
    if quant:
        q = torch.empty(y.shape, dtype=torch.int8, device=dev)
        scale = torch.empty(y.shape[:-1], dtype=torch.float32, device=dev)
    elif wn is not None:
        n = torch.empty(y.shape, dtype=y.dtype, device=dev)
    rstd = torch.empty(2, T, dtype=torch.float32, device=dev) if save else None
    _lib.check(_lib.lib().b200moe_block_norm(
        y2.data_ptr(), ys, _p(r2), rs, _p(w), _p(g2), gs, _p(wn), T, H, ROW_TYPES[y.dtype], _f32_bits(w, g2, wn), kind,
        alpha, eps, _p(h), _p(n), _p(q), _p(scale), _p(rstd), stream_of(y)), "block_norm")
    return h, n, q, scale, rstd


@functools.lru_cache(maxsize=256)
def _bwd_bytes(T, H, dt):
    b = ctypes.c_int64()
    _lib.check(_lib.lib().b200moe_block_norm_bwd_workspace(T, H, dt, ctypes.byref(b)), "block_norm_bwd_workspace")
    return b.value


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, gate, next_weight, kind, alpha, eps, want_h):
        with on_device(y):
            h, n, _, _, rstd = _forward(y, residual, weight, gate, kind, next_weight, alpha, eps, want_h, False, True)
        ctx.save_for_backward(y, residual, weight, gate, next_weight, rstd)
        ctx.kind, ctx.alpha = kind, alpha
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dn):
        y, residual, weight, gate, next_weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        with on_device(y):
            dev, H, dt = y.device, y.shape[-1], ROW_TYPES[y.dtype]
            y2, ys = rows_of(y)
            T = y2.shape[0]
            r2, rs = (None, 0) if residual is None else rows_of(residual)
            g2, gs = _gate_of(gate, ctx.kind)
            w = None if weight is None else weight.contiguous()
            wn = None if next_weight is None else next_weight.contiguous()
            dh = None if dh is None else dh.contiguous()
            dn = None if dn is None else dn.contiguous()

            def like(t, wanted):
                return torch.empty(t.shape, dtype=t.dtype, device=dev) if wanted else None

            dy, dr = like(y, need[0]), like(residual, need[1])
            dw, dg, dwn = like(weight, need[2]), like(gate, need[3]), like(next_weight, need[4])
            ws, size = None, 0
            if dw is not None or dwn is not None or (dg is not None and ctx.kind == _lib.GATE_CHANNEL):
                size = _bwd_bytes(T, H, dt)
                ws = torch.empty(size, dtype=torch.uint8, device=dev)
            _lib.check(_lib.lib().b200moe_block_norm_bwd(
                y2.data_ptr(), ys, _p(r2), rs, _p(w), _p(g2), gs, _p(wn), T, H, dt, _f32_bits(w, g2, wn), ctx.kind, ctx.alpha,
                rstd.data_ptr(), _p(dh), _p(dn), _p(dy), _p(dr), _p(dw), _p(dg), _p(dwn), _p(ws), size, stream_of(y)),
                "block_norm_bwd")
        return dy, dr, dw, dg, dwn, None, None, None, None


def _check(y, residual, weight, gate, next_weight, quant, what):
    if not y.is_cuda:
        raise RuntimeError(f"{what} runs on a CUDA device only (sm_100a); there is no CPU path")
    if y.dtype not in ROW_TYPES:
        raise TypeError("rows must be bfloat16, float16 or float32")
    H = y.shape[-1] if y.dim() else 0
    if not 1 <= H <= MAX_ROW:
        raise ValueError(f"rows must have 1 to {MAX_ROW} values")
    if quant not in (None, "int8"):
        raise ValueError(f"quant={quant!r}: None or 'int8'")
    if residual is not None and (residual.shape != y.shape or residual.dtype != y.dtype):
        raise ValueError("residual must have the rows' shape and type")
    for name, w in (("weight", weight), ("next_weight", next_weight)):
        if w is not None and (w.dim() != 1 or w.shape[0] != H or w.dtype not in (y.dtype, torch.float32)):
            raise ValueError(f"{name} must hold {H} values of the rows' type or float32")
    kind = _lib.GATE_NONE
    if gate is not None:
        if gate.dtype not in (y.dtype, torch.float32):
            raise TypeError("gate must be of the rows' type or float32")
        if gate.dim() == 1 and gate.shape[0] == H:
            kind = _lib.GATE_CHANNEL
        elif gate.shape == (*y.shape[:-1], 1):
            kind = _lib.GATE_TOKEN
        elif gate.shape == y.shape:
            kind = _lib.GATE_FULL
        else:
            raise ValueError(f"gate must be [{H}], [..., 1] or [..., {H}] over the rows' leading sizes")
    for t in (residual, weight, gate, next_weight):
        if t is not None and t.device != y.device:
            raise ValueError("all tensors must be on one device")
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, residual, weight, gate, next_weight))
    if grad and quant:
        raise RuntimeError("8-bit rows have no gradient: call it under torch.no_grad()")
    return kind, grad


def fused_pre_norm(x, weight, *, residual=None, eps=1e-6, quant=None):
    """Input norm of a block: n = h * rstd(h) * weight with h = x (+ residual), rstd(v) = 1 / sqrt(mean(v^2) + eps).

      ``x``, ``residual``: bf16, fp16 or fp32 [..., H], H <= 16384; rows may lie apart (views of wider tensors are read in place)
      ``weight``: [H], of the rows' type or float32
      ``quant="int8"``: n as 8-bit integers with one scale per token, for `linear_int8`; no gradient

    Arithmetic in 32 bits, each result rounded once; n is the norm of the unrounded sum.
    Returns n, or (q, scale) with ``quant``; with ``residual`` followed by h, the new residual stream."""
    if weight is None:
        raise ValueError("fused_pre_norm needs a weight")
    kind, grad = _check(x, residual, None, None, weight, quant, "fused_pre_norm")
    want_h = residual is not None
    if grad:
        h, n = _BlockNorm.apply(x, residual, None, None, weight, kind, 1.0, float(eps), want_h)
        return (n, h) if want_h else n
    with on_device(x):
        h, n, q, scale, _ = _forward(x, residual, None, None, kind, weight, 1.0, eps, want_h, quant, False)
    out = (q, scale) if quant else (n,)
    if want_h:
        out = (*out, h)
    return out if len(out) > 1 else n


def fused_post_norm(y, residual, weight=None, *, gate=None, residual_scale=1.0, eps=1e-6, next_weight=None, quant=None):
    """Output side of a block: h = residual_scale * residual + gate * u with u = y * rstd(y) * weight (u = y without weight),
    and with ``next_weight`` the next block's input norm n = h * rstd(h) * next_weight in the same launch.

      ``y``, ``residual``: bf16, fp16 or fp32 [..., H], H <= 16384
      ``gate``: [H] per channel, [..., 1] per token, or [..., H]; the rows' type or float32, as ``weight`` and ``next_weight`` [H]
      ``quant="int8"``: n as 8-bit integers with one scale per token, for `linear_int8`; no gradient

    Arithmetic in 32 bits, each result rounded once; n is the norm of the unrounded h.  Differentiable in all five tensors;
    gradients that sum over tokens are added in a fixed order.
    Returns h; (h, n) with ``next_weight``; (h, q, scale) with ``quant`` as well."""
    if residual is None:
        raise ValueError("fused_post_norm needs the residual")
    kind, grad = _check(y, residual, weight, gate, next_weight, quant, "fused_post_norm")
    if quant and next_weight is None:
        raise ValueError("quant belongs to the next block's input norm: pass next_weight")
    alpha = float(residual_scale)
    if grad:
        h, n = _BlockNorm.apply(y, residual, weight, gate, next_weight, kind, alpha, float(eps), True)
        return h if next_weight is None else (h, n)
    with on_device(y):
        h, n, q, scale, _ = _forward(y, residual, weight, gate, kind, next_weight, alpha, eps, True, quant, False)
    return (h, q, scale) if quant else h if next_weight is None else (h, n)
