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


_F32 = torch.float32


def _tensors(y, residual, weight, gate, kind, next_weight):
    """What the C calls take first: addresses and row distances of the inputs, the size, the types, the gate's kind.  Second: the
    tensors themselves, which may be copies and have to live until the launch."""
    y2, ys = rows_of(y)
    T, H = y2.shape
    r2 = g2 = None
    rs = gs = bits = 0
    if residual is not None:
        r2, rs = rows_of(residual)
    if weight is not None:
        weight = weight.contiguous()
        bits = weight.dtype is _F32
    if gate is not None:
        g2, gs = rows_of(gate) if kind == _lib.GATE_FULL else (gate.contiguous(), 1)
        bits |= (gate.dtype is _F32) << 1
    if next_weight is not None:
        next_weight = next_weight.contiguous()
        bits |= (next_weight.dtype is _F32) << 2
    return ((y2.data_ptr(), ys, None if r2 is None else r2.data_ptr(), rs, None if weight is None else weight.data_ptr(),
             None if g2 is None else g2.data_ptr(), gs, None if next_weight is None else next_weight.data_ptr(), T, H,
             ROW_TYPES[y.dtype], bits, kind), (y2, r2, weight, g2, next_weight))


def _forward(y, residual, weight, gate, kind, next_weight, alpha, eps, want_h, quant, save):
    args, _hold = _tensors(y, residual, weight, gate, kind, next_weight)
    h = torch.empty(y.shape, dtype=y.dtype, device=y.device) if want_h else None
    n = q = scale = rstd = None
    if quant:
        q = torch.empty(y.shape, dtype=torch.int8, device=y.device)
        scale = torch.empty(y.shape[:-1], dtype=_F32, device=y.device)
    elif next_weight is not None:
        n = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    if save:
        rstd = torch.empty(2 * args[8], dtype=_F32, device=y.device)
    _lib.check(_lib.lib().b200moe_block_norm(*args, alpha, eps, _p(h), _p(n), _p(q), _p(scale), _p(rstd),
                                             stream_of(y.get_device())), "block_norm")
    return h, n, q, scale, rstd


@functools.lru_cache(maxsize=256)
def _bwd_bytes(T, H, dt):
    b = ctypes.c_int64()
    _lib.check(_lib.lib().b200moe_block_norm_bwd_workspace(T, H, dt, ctypes.byref(b)), "block_norm_bwd_workspace")
    return b.value


def _backward(saved, need, how, dh, dn):
    y, residual, weight, gate, next_weight, rstd = saved
    kind, alpha = how
    args, _hold = _tensors(y, residual, weight, gate, kind, next_weight)
    if dh is not None:
        dh = dh.contiguous()
    if dn is not None:
        dn = dn.contiguous()
    dev = y.device
    dy, dr, dw, dg, dwn = (torch.empty(t.shape, dtype=t.dtype, device=dev) if w else None
                           for t, w in zip((y, residual, weight, gate, next_weight), need))
    ws, size = None, 0
    if dw is not None or dwn is not None or (dg is not None and kind == _lib.GATE_CHANNEL):
        size = _bwd_bytes(args[8], args[9], args[10])
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _lib.check(_lib.lib().b200moe_block_norm_bwd(
        *args, alpha, rstd.data_ptr(), _p(dh), _p(dn), _p(dy), _p(dr), _p(dw), _p(dg), _p(dwn), _p(ws), size,
        stream_of(y.get_device())), "block_norm_bwd")
    return dy, dr, dw, dg, dwn, None, None, None


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, gate, next_weight, how, eps, want_h):
        h, n, _, _, rstd = on_device(y.get_device(), _forward, y, residual, weight, gate, how[0], next_weight, how[1], eps, want_h,
                                     False, True)
        ctx.save_for_backward(y, residual, weight, gate, next_weight, rstd)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dn):
        saved = ctx.saved_tensors
        return on_device(saved[0].get_device(), _backward, saved, ctx.needs_input_grad, ctx.how, dh, dn)


def _check(y, residual, weight, gate, next_weight, quant, what):
    if not y.is_cuda:
        raise RuntimeError(f"{what} runs on a CUDA device only (sm_100a); there is no CPU path")
    dtype = y.dtype
    if dtype not in ROW_TYPES:
        raise TypeError("rows must be bfloat16, float16 or float32")
    shape = y.shape
    H = shape[-1] if shape else 0
    if not 1 <= H <= MAX_ROW:
        raise ValueError(f"rows must have 1 to {MAX_ROW} values")
    if quant is not None and quant != "int8":
        raise ValueError(f"quant={quant!r}: None or 'int8'")
    index = y.get_device()
    grad, away = y.requires_grad, False
    if residual is not None:
        if residual.dtype is not dtype or residual.shape != shape:
            raise ValueError("residual must have the rows' shape and type")
        grad |= residual.requires_grad
        away |= residual.get_device() != index
    for w in (weight, next_weight):
        if w is not None:
            if w.dim() != 1 or w.shape[0] != H or (w.dtype is not dtype and w.dtype is not _F32):
                raise ValueError(f"weights must hold {H} values of the rows' type or float32")
            grad |= w.requires_grad
            away |= w.get_device() != index
    kind = _lib.GATE_NONE
    if gate is not None:
        if gate.dtype is not dtype and gate.dtype is not _F32:
            raise TypeError("gate must be of the rows' type or float32")
        if gate.dim() == 1 and gate.shape[0] == H:
            kind = _lib.GATE_CHANNEL
        elif gate.shape == shape:
            kind = _lib.GATE_FULL
        elif gate.shape == (*shape[:-1], 1):
            kind = _lib.GATE_TOKEN
        else:
            raise ValueError(f"gate must be [{H}], [..., 1] or [..., {H}] over the rows' leading sizes")
        grad |= gate.requires_grad
        away |= gate.get_device() != index
    if away:
        raise ValueError("all tensors must be on one device")
    grad = grad and torch.is_grad_enabled()
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
        h, n = _BlockNorm.apply(x, residual, None, None, weight, (kind, 1.0), float(eps), want_h)
        return (n, h) if want_h else n
    h, n, q, scale, _ = on_device(x.get_device(), _forward, x, residual, None, None, kind, weight, 1.0, eps, want_h, quant, False)
    if quant:
        return (q, scale, h) if want_h else (q, scale)
    return (n, h) if want_h else n


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
        h, n = _BlockNorm.apply(y, residual, weight, gate, next_weight, (kind, alpha), float(eps), True)
        return h if next_weight is None else (h, n)
    h, n, q, scale, _ = on_device(y.get_device(), _forward, y, residual, weight, gate, kind, next_weight, alpha, eps, True, quant, False)
    return (h, q, scale) if quant else h if next_weight is None else (h, n)
