"""Router with what training it and watching its load need: `fused_topk`'s weights and ids, per-expert counts, the balance loss
and the z-loss from one pass over the logits, and the gradient of all of them (`b200moe_router_forward` two launches,
`b200moe_router_backward` one).  The reference takes ids and weights from outside its operator
(tests/contrib/moe/test_moe_sorting.py:81-84) and has no counterpart of the losses.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class RouterOutput(NamedTuple):
    topk_weights: torch.Tensor     # f32 [T, K]
    topk_ids: torch.Tensor         # i32 [T, K]
    counts: torch.Tensor           # i32 [E], or [sequences, E] with cu_seqlens
    balance_loss: torch.Tensor     # f32 scalar
    z_loss: torch.Tensor           # f32 scalar


def fused_router(gating_output, topk: int, *, renormalize: bool = True, scoring: str = "softmax", token_mask=None,
                 cu_seqlens=None) -> RouterOutput:
    """Top-k routing with per-expert counts, balance loss and z-loss, differentiable in the logits (in reverse mode and once;
    forward-mode derivatives and tracing are refused).

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
    return RouterOutput(*_lib.dense().router(gating_output, topk, renormalize, scoring, token_mask, cu_seqlens))
