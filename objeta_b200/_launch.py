"""Where a call on torch tensors runs: its device made current, its stream, and
the tensors that the call makes allocated for that stream."""
from __future__ import annotations

import contextlib


class _Here:
    """The current device already fits: nothing to change."""
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


_raw_stream = None  # device index -> handle of torch's current stream


def _raw_stream_getter():
    """torch's own getter of the raw handle where it has one (a tenth of the
    time of building a Stream object), else the public one."""
    global _raw_stream
    import torch
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                          lambda index: torch.cuda.current_stream(index).cuda_stream)
    return _raw_stream


def launch(device, stream=None):
    """A context whose value is the stream's handle: ``stream`` (a torch stream
    or a handle), or the current torch stream of ``device``.  Inside it
    ``device`` is current and new tensors belong to the stream."""
    import torch
    index = device.index
    if stream is None and torch.cuda.current_device() == index:
        return _Here((_raw_stream or _raw_stream_getter())(index))
    return _there(device, stream)


def _refuse(name, t, device, dtypes, shape, contiguous):
    import torch
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
        ok = t.is_cuda
        dev = t.device
    except AttributeError:
        ok = False
    if not ok or (device is not None and dev != device) or (dtypes is not None and t.dtype not in dtypes) or (
            shape is not None and t.shape != shape) or (contiguous and not t.is_contiguous()):
        _refuse(name, t, device, dtypes, shape, contiguous)
    return dev


def matrix(name, t, device=None, dtypes=None, shape=None):
    """Checks a 2-D tensor argument whose rows are contiguous (the rows may lie
    apart); returns (rows, cols, elements between rows)."""
    on_device(name, t, device, dtypes, shape, False)
    size = t.shape
    if len(size) == 2:
        rows, cols = size
        if t.is_contiguous():
            return rows, cols, cols
        down, along = t.stride()
        if (cols <= 1 or along == 1) and (rows <= 1 or down >= cols):
            return rows, cols, down if rows > 1 else cols
    raise ValueError(f"{name}: expected rows of contiguous elements, got strides {t.stride()} of {tuple(size)}")
