"""Where a call on torch tensors runs: its device made current, its stream, and
the tensors that the call makes allocated for that stream."""
from __future__ import annotations

import contextlib

import torch


# torch's own getters of the current device and of the raw handle of its
# current stream where it has them (a fraction of the time of the public ones,
# which build objects), else the public ones
current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                     lambda index: torch.cuda.current_stream(index).cuda_stream)


@contextlib.contextmanager
def launch(device, stream=None):
    """A context whose value is the stream's handle: ``stream`` (a torch stream
    or a handle), or the current torch stream of ``device``.  Inside it
    ``device`` is current and new tensors belong to the stream."""
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
            return
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
        if getattr(stream, "cuda_stream", None) is None:
            raise TypeError(f"cannot use {stream!r} as a CUDA stream")
        if stream.device != device:
            raise ValueError(f"the stream is of {stream.device}, the tensors are on {device}")
        with torch.cuda.stream(stream):
            yield stream.cuda_stream


def run(device, stream, fn, *args):
    """fn(stream handle, *args) inside ``launch``; directly where the current
    device and stream already fit."""
    if stream is None and device.index == current_device():
        return fn(raw_stream(device.index), *args)
    with launch(device, stream) as st:
        return fn(st, *args)


def _refuse(name, t, device, dtypes, shape, contiguous):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors are on {device}")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name} is {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")


def on_device(name, t, device=None, dtypes=None, shape=None, contiguous=True):
    """Checks one tensor argument; returns its device."""
    try:
        dev = t.device
    except AttributeError:
        dev = None
    if dev is None or (dev.type != "cuda" if device is None else dev != device) or (
            dtypes is not None and t.dtype not in dtypes) or (shape is not None and t.shape != shape) or (
            contiguous and not t.is_contiguous()):
        _refuse(name, t, device, dtypes, shape, contiguous)
    return dev


def matrix(name, t, device=None, dtypes=None, shape=None):
    """Checks a 2-D tensor argument whose rows are contiguous (the rows may lie
    apart); returns (rows, cols, elements between rows)."""
    try:
        size, dev = t.shape, t.device
    except AttributeError:
        size = dev = None
    if dev is None or (dev.type != "cuda" if device is None else dev != device) or (
            dtypes is not None and t.dtype not in dtypes) or (shape is not None and size != shape):
        _refuse(name, t, device, dtypes, shape, False)
    if len(size) == 2:
        rows, cols = size
        if t.is_contiguous():
            return rows, cols, cols
        down, along = t.stride()
        if (cols <= 1 or along == 1) and (rows <= 1 or down >= cols):
            return rows, cols, down if rows > 1 else cols
    raise ValueError(f"{name}: expected rows of contiguous elements, got strides {t.stride()} of {tuple(size)}")
