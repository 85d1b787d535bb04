"""Router with what training it and watching its load need: `fused_topk`'s weights and ids, per-expert counts, the balance loss
and the z-loss from one pass over the logits, and the gradient of all of them (`b200moe_router_forward` two launches,
`b200moe_router_backward` one).  The reference takes ids and weights from outside its operator
(tests/contrib/moe/test_moe_sorting.py:81-84) and has no counterpart of the losses.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rows import ROW_TYPES, on_device, rows_of, stream_of

MAX_EXPERTS, MAX_TOPK = 1024, 32
_SCORING = {"softmax": 0, "sigmoid": 1}


class RouterOutput(NamedTuple):
    topk_weights: torch.Tensor     # f32 [T, K]
    topk_ids: torch.Tensor         # i32 [T, K]
    counts: torch.Tensor           # i32 [E], or [sequences, E] with cu_seqlens
    balance_loss: torch.Tensor     # f32 scalar
    z_loss: torch.Tensor           # f32 scalar


@functools.lru_cache(maxsize=256)
def _layout(T, E, S):
    """Byte sizes: the launch's workspace; what the backward pass needs (lse [2, T], seg [T], coef [S, E], stats [2] in a row)."""
    b = ctypes.c_int64()
    _lib.check(_lib.lib().b200moe_router_workspace(T, E, S, ctypes.byref(b)), "router_workspace")
    return b.value, 4 * (3 * T + S * E + 2)


def _p(t):
    return None if t is None else t.data_ptr()


def _saved_at(saved, T, S, E):
    lse = saved.data_ptr()
    return lse, lse + 8 * T, lse + 12 * T, lse + 12 * T + 4 * S * E


def _forward(logits, K, scoring, renorm, mask, cu, save):
    x, stride = rows_of(logits)
    T, E = x.shape
    dev = x.device
    S = 1 if cu is None else cu.shape[0] - 1
    work, keep = _layout(T, E, S)
    weights = torch.empty((T, K), dtype=torch.float32, device=dev)
    ids = torch.empty((T, K), dtype=torch.int32, device=dev)
    counts = torch.empty((E,) if cu is None else (S, E), dtype=torch.int32, device=dev)
    balance = torch.empty((), dtype=torch.float32, device=dev)
    z = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(work, dtype=torch.uint8, device=dev)
    saved, at = None, (None, None, None, None)
    if save:
        saved = torch.empty(keep, dtype=torch.uint8, device=dev)
        at = _saved_at(saved, T, S, E)
    _lib.check(_lib.lib().b200moe_router_forward(
        x.data_ptr(), stride, T, E, K, ROW_TYPES[x.dtype], scoring, renorm, _p(mask), _p(cu), S, weights.data_ptr(),
        ids.data_ptr(), counts.data_ptr(), balance.data_ptr(), z.data_ptr(), *at, ws.data_ptr(), work,
        stream_of(x.get_device())), "router_forward")
    return weights, ids, counts, balance, z, saved


def _backward(logits, weights, ids, saved, how, dweights, dbalance, dz):
    K, scoring, renorm, S = how
    x, stride = rows_of(logits)
    T, E = x.shape
    if dweights is not None:
        dweights = dweights.contiguous()
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _lib.check(_lib.lib().b200moe_router_backward(
        x.data_ptr(), stride, T, E, K, ROW_TYPES[x.dtype], scoring, renorm, *_saved_at(saved, T, S, E), ids.data_ptr(),
        weights.data_ptr(), _p(dweights), _p(dbalance), _p(dz), out.data_ptr(), stream_of(x.get_device())), "router_backward")
    return out, None, None, None, None, None


class _Router(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, K, scoring, renorm, mask, cu):
        weights, ids, counts, balance, z, saved = on_device(logits.get_device(), _forward, logits, K, scoring, renorm, mask, cu, True)
        # the rows that the backward pass reads are the input itself: saved as such, so that a change in place is noticed
        ctx.save_for_backward(logits, weights, ids, saved)
        ctx.how = (K, scoring, renorm, 1 if cu is None else cu.shape[0] - 1)
        ctx.mark_non_differentiable(ids, counts)
        ctx.set_materialize_grads(False)
        return weights, ids, counts, balance, z

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _ids, _counts, dbalance, dz):
        logits, weights, ids, saved = ctx.saved_tensors
        return on_device(logits.get_device(), _backward, logits, weights, ids, saved, ctx.how, dweights, dbalance, dz)


def fused_router(gating_output, topk: int, *, renormalize: bool = True, scoring: str = "softmax", token_mask=None,
                 cu_seqlens=None) -> RouterOutput:
    """Top-k routing with per-expert counts, balance loss and z-loss, differentiable in the logits.

      ``gating_output``: logits [T, E], bf16, fp16 or fp32, E <= 1024; rows may lie apart
      ``topk``: experts per token, up to 32; the largest LOGITS, equal ones in ascending order
      ``renormalize``: divide a token's weights by their sum;  ``scoring``: "softmax" or "sigmoid"
      ``token_mask``: bool [T], False = padding
      ``cu_seqlens``: int32 [S+1], ascending from 0 or later to T at most: token t is in sequence s if
        cu_seqlens[s] <= t < cu_seqlens[s+1].  The balance loss is then the mean over the sequences that hold tokens.  Its
        values are read on the device only; values out of order give wrong sums, never an access out of range.

    A token that is masked, in no sequence, or has only -inf logits takes part in nothing: ids 0..K-1, weights 0, no gradient,
    whatever its logits hold.  With n_s live tokens in sequence s, p = softmax(logits) or sigmoid(logits) / their sum:
      balance_loss = mean_s  E / (K n_s^2) * sum_e counts[s, e] * sum_t p[t, e]      (1 when the load is even)
      z_loss = mean over the live tokens of logsumexp(logits)^2
    Both are 0 without live tokens; counts take no gradient.  The same bits on every run."""
    if not gating_output.is_cuda:
        raise RuntimeError("fused_router runs on a CUDA device only (sm_100a); there is no CPU path")
    if gating_output.dtype not in ROW_TYPES:
        raise TypeError("gating_output must be bfloat16, float16 or float32")
    if gating_output.dim() != 2:
        raise ValueError("gating_output must be [T, E]")
    T, E = gating_output.shape
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"{E} experts: 1 to {MAX_EXPERTS} are supported")
    if not 1 <= topk <= min(E, MAX_TOPK):
        raise ValueError(f"topk={topk}: 1 to {min(E, MAX_TOPK)} for {E} experts")
    if scoring not in _SCORING:
        raise ValueError(f"scoring={scoring!r}: 'softmax' or 'sigmoid'")
    if token_mask is not None:
        if token_mask.dtype != torch.bool or token_mask.shape != (T,) or token_mask.device != gating_output.device:
            raise ValueError("token_mask must be a bool tensor [T] on the logits' device")
        token_mask = token_mask.contiguous()
    if cu_seqlens is not None:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2 or cu_seqlens.device != gating_output.device:
            raise ValueError("cu_seqlens must be an int32 tensor [S+1] on the logits' device")
        cu_seqlens = cu_seqlens.contiguous()
    args = (int(topk), _SCORING[scoring], 1 if renormalize else 0, token_mask, cu_seqlens)
    if gating_output.requires_grad and torch.is_grad_enabled():
        return RouterOutput(*_Router.apply(gating_output, *args))
    return RouterOutput(*on_device(gating_output.get_device(), _forward, gating_output, *args, False)[:5])
