"""RMS norms on both sides of a transformer block, fused with what stands next to them: the branch's gate, the residual sum
and its scale, and the 8-bit rows that `linear_int8` takes.  One launch forward (`b200moe_block_norm`), two backward
(`b200moe_block_norm_bwd`; one where no parameter takes a gradient).  The reference has no counterpart: its MoE operator starts
behind the norm and ends before the residual sum.
"""
from __future__ import annotations

import torch

from . import _lib


def _number(v, name):
    """v as a plain number.  Nothing flows back into it, so a parameter in its place would train without a gradient."""
    if not isinstance(v, torch.Tensor):
        return v
    if (v.requires_grad and torch.is_grad_enabled()) or torch.autograd.forward_ad.unpack_dual(v).tangent is not None:
        raise RuntimeError(f"{name} is a number and has no gradient: fold a learned factor into the weight or the gate, or scale the residual itself")
    return v.detach()


def fused_pre_norm(x, weight, *, residual=None, eps=1e-6, quant=None):
    """Input norm of a block: n = h * rstd(h) * weight with h = x (+ residual), rstd(v) = 1 / sqrt(mean(v^2) + eps).

      ``x``, ``residual``: bf16, fp16 or fp32 [..., H], H <= 16384; rows may lie apart (views of wider tensors are read in place)
      ``weight``: [H], of the rows' type or float32
      ``quant="int8"``: n as 8-bit integers with one scale per token, for `linear_int8`; no gradient

    Arithmetic in 32 bits, each result rounded once; n is the norm of the unrounded sum.  Differentiable as `fused_post_norm`.
    Returns n, or (q, scale) with ``quant``; with ``residual`` followed by h, the new residual stream."""
    if weight is None:
        raise ValueError("fused_pre_norm needs a weight")
    if quant is not None and quant != "int8":
        raise ValueError(f"quant={quant!r}: None or 'int8'")
    out = _lib.dense().block_norm(x, residual, None, None, weight, 1.0, _number(eps, "eps"), residual is not None, quant is not None, "fused_pre_norm")
    if residual is None:
        return out[0] if quant is None else tuple(out)
    return (*out[1:], out[0])


def fused_post_norm(y, residual, weight=None, *, gate=None, residual_scale=1.0, eps=1e-6, next_weight=None, quant=None):
    """Output side of a block: h = residual_scale * residual + gate * u with u = y * rstd(y) * weight (u = y without weight),
    and with ``next_weight`` the next block's input norm n = h * rstd(h) * next_weight in the same launch.

      ``y``, ``residual``: bf16, fp16 or fp32 [..., H], H <= 16384
      ``gate``: [H] per channel, [..., 1] per token, or [..., H]; the rows' type or float32, as ``weight`` and ``next_weight`` [H]
      ``residual_scale``: a number; it takes no gradient, and a tensor that asks for one is refused
      ``quant="int8"``: n as 8-bit integers with one scale per token, for `linear_int8`; no gradient

    Arithmetic in 32 bits, each result rounded once; n is the norm of the unrounded h.  Differentiable in all five tensors, in
    reverse mode and once; forward-mode derivatives and tracing are refused.  Gradients that sum over tokens are added in a fixed
    order.  A row's sum of squares is a 32-bit number too: an RMS of more than 1.8e19 / sqrt(H) makes its rstd 0, as in torch.
    Returns h; (h, n) with ``next_weight``; (h, q, scale) with ``quant`` as well."""
    if residual is None:
        raise ValueError("fused_post_norm needs the residual")
    if quant is not None:
        if quant != "int8":
            raise ValueError(f"quant={quant!r}: None or 'int8'")
        if next_weight is None:
            raise ValueError("quant belongs to the next block's input norm: pass next_weight")
    out = _lib.dense().block_norm(y, residual, weight, gate, next_weight, _number(residual_scale, "residual_scale"), _number(eps, "eps"), True,
                                  quant is not None, "fused_post_norm")
    return out[0] if next_weight is None else tuple(out)
