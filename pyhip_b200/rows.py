"""What the row-wise operators share: element types, rows of strided tensors, the current device and stream.

Decode-sized calls of these operators take a few microseconds on the GPU, less than a handful of Python calls: the helpers
here and their callers look things up once and in the cheapest way torch offers."""
from __future__ import annotations

import torch

from . import _lib

ROW_TYPES = {torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_FP16, torch.float32: _lib.T_FP32}
MAX_ROW = 16384            # values of a row that the row-wise kernels hold in registers

current_device = torch.cuda.current_device
if hasattr(torch._C, "_cuda_getDevice"):
    current_device = torch._C._cuda_getDevice


def stream_of(index):
    """Handle of the current stream on device ``index``."""
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):          # the same without building a Stream object (2 us)
    stream_of = torch._C._cuda_getCurrentRawStream


def on_device(index, call, *args):
    """``call(*args)`` with device ``index`` current: launches go to the current device."""
    if index == current_device():
        return call(*args)
    with torch.cuda.device(index):
        return call(*args)


def rows_of(x):
    """``x`` [..., H] as ([T, H] with neighbouring values adjacent, elements between its rows): a view wherever one exists."""
    if x.is_contiguous():
        H = x.shape[-1]
        return (x if x.dim() == 2 else x.view(x.numel() // H if H else 0, H)), H
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1]) if x.numel() else x.new_empty((x.shape[:-1].numel(), x.shape[-1]))
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])
