"""What the operators' Python entry points share: argument checks, the device
and stream a call runs on, and its workspace."""
from __future__ import annotations

import contextlib

import torch

from . import _check, load

_current = contextlib.nullcontext()
_scratch: dict = {}
_sizes: dict = {}
_raw_stream = torch._C._cuda_getCurrentRawStream
_COUNTERS = 4096  # arrival counters at the start of a workspace, zero between launches


def want(t, name: str, dtype, shape=None, device=None):
    """`t` is a CUDA tensor of `dtype` (or one of them) and `shape` on `device`."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype if isinstance(dtype, torch.dtype) else t.dtype not in dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def want_out(t, name: str, dtype, shape, device):
    """As `want`, for a tensor whose memory is used as it lies: contiguous as well."""
    want(t, name, dtype, shape, device)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def on(device, stream, *used):
    """The context a call runs in: `device` current and `stream` (None: the
    device's current one) the stream, so that what the call allocates belongs
    to it. Tensors in `used` are marked as used on an explicit stream."""
    if stream is None:
        if device.index == torch.cuda.current_device():
            return _current
        return torch.cuda.device(device)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device)
    elif stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
    for t in used:
        if t is not None:
            t.record_stream(stream)
    return torch.cuda.stream(stream)


def run(name: str, device, *args) -> None:
    """Calls entry point `name` on `device`'s current stream (its last argument)."""
    status = getattr(load(), name)(*args, _raw_stream(device.index))
    if status != 0:
        _check(name, status)


def size(query, device, *key) -> int:
    """A workspace size query, remembered: a pure function of the device and the sizes."""
    key = (query, device.index, *key)
    n = _sizes.get(key)
    if n is None:
        if len(_sizes) > 4096:  # calls of ever new sizes do not fill the memory
            _sizes.clear()
        n = _sizes[key] = query(*key[2:])
    return n


def workspace(need: int, device):
    """A workspace of at least `need` bytes with zeroed arrival counters for a
    launch on the current stream; None for 0.

    Calls on one stream share a buffer (their order keeps it theirs alone).
    While the stream is being captured into a graph each call takes its own
    from the graph's memory and clears its counters in the graph, so graphs
    share nothing with each other or with eager calls."""
    if need == 0:
        return None
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:_COUNTERS].zero_()
        return ws
    key = (device.index, _raw_stream(device.index))
    ws = _scratch.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:_COUNTERS].zero_()
        _scratch[key] = ws
    return ws
