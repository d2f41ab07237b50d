"""Stream and device handling of calls that are short enough for its cost to count.

`torch.cuda.current_stream()` builds a Stream object per call and `torch.cuda.device` switches back and forth even
where the device is the current one already; both cost as much as a small kernel's launch.
"""
from __future__ import annotations

import contextlib

import torch

_streams: dict[tuple[int, int], torch.cuda.Stream] = {}
_STAY = contextlib.nullcontext()


def on_device(device: torch.device):
    """Context in which `device` is the current one."""
    return _STAY if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_of(device: torch.device, *tensors) -> int:
    """Handle of the device's current stream, for a launch that reads `tensors` (None allowed): their storage is kept
    until that stream has read it, also where they were made on another one."""
    handle = torch._C._cuda_getCurrentRawStream(device.index)
    stream = _streams.get((device.index, handle))
    if stream is None:
        stream = _streams[device.index, handle] = torch.cuda.current_stream(device)
    for tensor in tensors:
        if tensor is not None:
            tensor.record_stream(stream)
    return handle
