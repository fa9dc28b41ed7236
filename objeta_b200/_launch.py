"""Where a call on torch tensors runs: its device made current, its stream, and
the tensors that the call makes allocated for that stream."""
from __future__ import annotations

import contextlib


class _Here:
    """The current device and stream already fit: nothing to change."""
    __slots__ = ("handle",)

    def __init__(self, handle):
        self.handle = handle

    def __enter__(self):
        return self.handle

    def __exit__(self, *exc):
        return False


@contextlib.contextmanager
def _there(device, stream):
    import torch
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


def launch(device, stream=None):
    """A context whose value is the stream's handle: ``stream`` (a torch stream
    or a handle), or the current torch stream of ``device``.  Inside it
    ``device`` is current and new tensors belong to the stream."""
    import torch
    if stream is None and torch.cuda.current_device() == device.index:
        return _Here(torch.cuda.current_stream().cuda_stream)
    return _there(device, stream)


def on_device(name, t, device=None, dtypes=None, shape=None, contiguous=True):
    """Checks one tensor argument; returns its device."""
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors are on {device}")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name} is {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")
    return t.device


def row_stride(name, t):
    """Elements between the rows of a 2-D tensor whose rows are contiguous."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name}: expected rows of contiguous elements, got strides {t.stride()} of {tuple(t.shape)}")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]
