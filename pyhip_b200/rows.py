"""What the row-wise operators share: element types, rows of strided tensors, the current device and stream."""
from __future__ import annotations

import contextlib

import torch

from . import _lib

ROW_TYPES = {torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_FP16, torch.float32: _lib.T_FP32}
MAX_ROW = 16384            # values of a row that the row-wise kernels hold in registers
_here = contextlib.nullcontext()


def on_device(x):
    """Makes ``x``'s device the current one (launches go to the current device)."""
    return _here if x.device.index == torch.cuda.current_device() else torch.cuda.device(x.device)


def stream_of(x):
    """Handle of the current stream on ``x``'s device."""
    return torch.cuda.current_stream(x.device).cuda_stream


def rows_of(x):
    """``x`` [..., H] as ([T, H] with neighbouring values adjacent, elements between its rows): a view wherever one exists."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty((x.shape[:-1].numel(), x.shape[-1]))
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])
