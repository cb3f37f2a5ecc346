"""What the operators' Python entry points share: the device and stream a call
runs on, and the module that checks its tensors and makes the call."""
from __future__ import annotations

import contextlib
import functools
import os

import torch

from . import HERE, load

_current = contextlib.nullcontext()
_binding = None


def binding():
    """The compiled host path (csrc/binding.cpp), built beside libi4g.so."""
    global _binding
    if _binding is None:
        load()  # names what is missing where nothing is built
        if not os.path.exists(os.path.join(HERE, "_binding.so")):
            raise ImportError(f"{HERE}/_binding.so is not built; run `make -C {HERE} python`")
        from . import _binding as module
        if not torch.__version__.startswith(module.torch_version):
            raise ImportError(f"_binding.so was built against torch {module.torch_version}, not "
                              f"{torch.__version__}; run `make -C {HERE} python`")
        _binding = module
    return _binding


def cuda_device(t, name: str) -> torch.device:
    """The device of `t`, which must be a CUDA tensor."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    return t.device


def on(device, stream, *used):
    """The context a call runs in: `device` current and `stream` (None: the
    device's current one) the stream, so that what the call allocates belongs
    to it. Tensors in `used` are marked as used on an explicit stream."""
    if stream is None:
        if device.index == torch.cuda.current_device():
            return _current
        return torch.cuda.device(device)
    return torch.cuda.stream(mark(device, stream, *used))


@functools.lru_cache(maxsize=64)
def _external(handle: int, device) -> torch.cuda.Stream:
    return torch.cuda.ExternalStream(handle, device=device)


def mark(device, stream, *used) -> torch.cuda.Stream:
    """Marks the tensors in `used` as used on the explicit `stream`, which it returns."""
    if isinstance(stream, int):
        stream = _external(stream, device)
    elif stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
    for t in used:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            t.record_stream(stream)
    return stream
