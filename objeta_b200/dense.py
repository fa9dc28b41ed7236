"""Dense products of many tokens: ``linear`` with bias, activation and residual
in its epilogue, its gradients, and the shared expert of a batch.

The reference's dense paths run one token (``gemv_bf16_device``,
``ffn_bf16_device``); these take T of them: the router's projection, the
shared expert beside ``moe_pairs``, an output head.  Types: x and w both bf16,
both f16, x f32 with w bf16, or both f32; y f32 or, where x is a 16-bit type,
that type.  Any sizes, row strides and element-aligned addresses.
"""
from __future__ import annotations

import ctypes

from . import _lib
from ._launch import launch, on_device, row_stride

c_size = ctypes.c_size_t
c_int = ctypes.c_int
c_int32 = ctypes.c_int32
c_float = ctypes.c_float
c_void_p = ctypes.c_void_p

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_DX, _DW, _DBIAS = 1, 2, 4


class _LinearDesc(ctypes.Structure):
    _fields_ = ([(n, c_size) for n in ("tokens", "in_features", "out_features")]
                + [(n, c_int32) for n in ("x_dtype", "w_dtype", "y_dtype", "bias_dtype", "activation", "reserved")]
                + [(n, c_size) for n in ("x_stride", "w_stride", "y_stride", "residual_stride", "z_stride")])


class _LinearBackwardDesc(ctypes.Structure):
    _fields_ = ([(n, c_size) for n in ("tokens", "in_features", "out_features")]
                + [(n, c_int32) for n in ("x_dtype", "w_dtype", "dy_dtype", "dw_dtype", "activation", "outputs",
                                          "accumulate", "reserved")]
                + [(n, c_size) for n in ("dy_stride", "z_stride", "x_stride", "w_stride", "dx_stride", "dw_stride")])


_lib.register_signatures({
    "objb_linear_scratch_bytes": (c_int, [c_void_p, c_void_p, c_void_p, ctypes.POINTER(c_size)]),
    "objb_linear_device": (c_int, [c_void_p] * 8 + [c_size, c_void_p]),
    "objb_linear_backward_scratch_bytes": (c_int, [c_void_p] * 4 + [ctypes.POINTER(c_size)]),
    "objb_linear_backward_device": (c_int, [c_void_p] * 9 + [c_size, c_void_p]),
    "objb_ffn_bf16_tokens_scratch_bytes": (c_int, [c_void_p] * 3 + [c_size] * 4 + [ctypes.POINTER(c_size)]),
    "objb_ffn_bf16_tokens_device": (c_int, [c_void_p, c_void_p, c_void_p, c_size, c_size, c_size, c_void_p, c_size,
                                            c_void_p, c_void_p, c_float, c_void_p, c_size, c_void_p]),
})

_codes = None


def _dtype_code(name, dtype):
    global _codes
    if _codes is None:
        import torch
        _codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    if dtype not in _codes:
        raise ValueError(f"{name} is {dtype}, expected torch.float32, torch.float16 or torch.bfloat16")
    return _codes[dtype]


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}, expected one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def _p(t):
    return t.data_ptr() if t is not None else None


def _rows(name, t, device, shape=None):
    on_device(name, t, device, shape=shape, contiguous=False)
    return row_stride(name, t)


def _scratch(call, device, *args):
    import torch
    n = c_size()
    _lib.call(call, *args, ctypes.byref(n))
    return torch.empty(int(n.value), dtype=torch.uint8, device=device) if n.value else None


def linear(d_x, d_w, d_bias=None, activation: str = "none", d_residual=None, out_dtype=None, d_y=None, d_z=None,
           stream=None):
    """y = act(d_x d_w^T + d_bias) + d_residual.

    d_x [T, in], d_w [out, in], d_bias [out] (f32 or d_w's type), d_residual
    [T, out] of y's type (may be ``d_y`` itself).  ``activation``: "none",
    "relu", "silu", "gelu" (erf) or "gelu_tanh".  ``out_dtype`` defaults to
    d_x's type.  ``d_z`` [T, out], of y's type, receives d_x d_w^T + d_bias for
    ``linear_backward``.
    """
    import torch
    dev = on_device("d_x", d_x, contiguous=False)
    ldx = _rows("d_x", d_x, dev)
    T, K = d_x.shape
    ldw = _rows("d_w", d_w, dev)
    N = d_w.shape[0]
    if d_w.shape[1] != K:
        raise ValueError(f"d_w has shape {tuple(d_w.shape)}, expected (out, {K})")
    with launch(dev, stream) as st:
        if d_y is None:
            d_y = torch.empty(T, N, dtype=out_dtype or d_x.dtype, device=dev)
        elif out_dtype is not None and d_y.dtype != out_dtype:
            raise ValueError(f"d_y is {d_y.dtype}, out_dtype {out_dtype}")
        d = _LinearDesc(tokens=T, in_features=K, out_features=N, x_dtype=_dtype_code("d_x", d_x.dtype),
                        w_dtype=_dtype_code("d_w", d_w.dtype), y_dtype=_dtype_code("d_y", d_y.dtype),
                        activation=_activation(activation), x_stride=ldx, w_stride=ldw,
                        y_stride=_rows("d_y", d_y, dev, (T, N)))
        if d_bias is not None:
            on_device("d_bias", d_bias, dev, shape=(N,))
            d.bias_dtype = _dtype_code("d_bias", d_bias.dtype)
        if d_residual is not None:
            on_device("d_residual", d_residual, dev, (d_y.dtype,), contiguous=False)
            d.residual_stride = _rows("d_residual", d_residual, dev, (T, N))
        if d_z is not None:
            on_device("d_z", d_z, dev, (d_y.dtype,), contiguous=False)
            d.z_stride = _rows("d_z", d_z, dev, (T, N))
        ref = ctypes.byref(d)
        scratch = _scratch("objb_linear_scratch_bytes", dev, ref, d_x.data_ptr(), d_w.data_ptr())
        _lib.call("objb_linear_device", ref, d_x.data_ptr(), d_w.data_ptr(), _p(d_bias), _p(d_residual),
                  d_y.data_ptr(), _p(d_z), _p(scratch), scratch.numel() if scratch is not None else 0, st)
    return d_y


def linear_backward(d_dy, d_x, d_w, d_z=None, activation: str = "none", need_dx: bool = True, need_dw: bool = True,
                    need_dbias: bool = False, dw_dtype=None, d_dx=None, d_dw=None, d_dbias=None,
                    accumulate: bool = False, stream=None):
    """The gradients (dx, dw, dbias) of ``linear`` from d_dy [T, out]; those not
    needed are None.

    ``d_z``: the one ``linear`` kept (of d_dy's type; only read with an
    activation).  dx has d_x's type, dw d_w's type or f32 (``dw_dtype``), dbias
    f32.  ``accumulate`` adds to the given d_dw and d_dbias.  The residual's
    gradient is d_dy.  Under a 16-bit d_dy, dy act'(z) enters the two products
    rounded to that type unless dw is f32; dbias sums it unrounded.
    """
    import torch
    dev = on_device("d_dy", d_dy, contiguous=False)
    lddy = _rows("d_dy", d_dy, dev)
    T, N = d_dy.shape
    ldw = _rows("d_w", d_w, dev)
    if d_w.shape[0] != N:
        raise ValueError(f"d_w has shape {tuple(d_w.shape)}, expected ({N}, in)")
    K = d_w.shape[1]
    ldx = _rows("d_x", d_x, dev, (T, K))
    act = _activation(activation)
    if act and d_z is None:
        raise ValueError(f"the gradient of {activation!r} needs d_z")
    if accumulate and ((need_dw and d_dw is None) or (need_dbias and d_dbias is None)):
        raise ValueError("accumulate needs the d_dw and d_dbias to add to")
    with launch(dev, stream) as st:
        if need_dx:
            if d_dx is None:
                d_dx = torch.empty(T, K, dtype=d_x.dtype, device=dev)
            else:
                on_device("d_dx", d_dx, dev, (d_x.dtype,), contiguous=False)
        if need_dw:
            if d_dw is None:
                d_dw = torch.empty(N, K, dtype=dw_dtype or d_w.dtype, device=dev)
            elif dw_dtype is not None and d_dw.dtype != dw_dtype:
                raise ValueError(f"d_dw is {d_dw.dtype}, dw_dtype {dw_dtype}")
        if need_dbias:
            if d_dbias is None:
                d_dbias = torch.empty(N, dtype=torch.float32, device=dev)
            else:
                on_device("d_dbias", d_dbias, dev, (torch.float32,), (N,))
        d = _LinearBackwardDesc(tokens=T, in_features=K, out_features=N, x_dtype=_dtype_code("d_x", d_x.dtype),
                                w_dtype=_dtype_code("d_w", d_w.dtype), dy_dtype=_dtype_code("d_dy", d_dy.dtype),
                                dw_dtype=_dtype_code("d_dw", d_dw.dtype if need_dw else d_w.dtype), activation=act,
                                outputs=_DX * bool(need_dx) | _DW * bool(need_dw) | _DBIAS * bool(need_dbias),
                                accumulate=int(bool(accumulate)), dy_stride=lddy, x_stride=ldx, w_stride=ldw)
        if act:
            on_device("d_z", d_z, dev, (d_dy.dtype,), contiguous=False)
            d.z_stride = _rows("d_z", d_z, dev, (T, N))
        if need_dx:
            d.dx_stride = _rows("d_dx", d_dx, dev, (T, K))
        if need_dw:
            d.dw_stride = _rows("d_dw", d_dw, dev, (N, K))
        ref = ctypes.byref(d)
        scratch = _scratch("objb_linear_backward_scratch_bytes", dev, ref, d_dy.data_ptr(), d_x.data_ptr(),
                           d_w.data_ptr())
        _lib.call("objb_linear_backward_device", ref, d_dy.data_ptr(), _p(d_z) if act else None, d_x.data_ptr(),
                  d_w.data_ptr(), _p(d_dx) if need_dx else None, _p(d_dw) if need_dw else None,
                  _p(d_dbias) if need_dbias else None, _p(scratch), scratch.numel() if scratch is not None else 0, st)
    return d_dx if need_dx else None, d_dw if need_dw else None, d_dbias if need_dbias else None


def ffn_bf16_tokens(d_gate, d_up, d_down, d_x, d_residual=None, d_out=None, swiglu_limit: float = 0.0, stream=None):
    """``ffn_bf16_device`` for T tokens (the shared expert of a batch):
    out[t] = d_residual[t] + down SwiGLU(gate x_t, up x_t).

    d_gate, d_up [I, H] and d_down [O, I] bf16, d_x f32 [T, H], d_residual f32
    [T, O] or None; ``d_out`` may be ``d_residual`` itself.  f32 precision
    throughout, as the one-token call.
    """
    import torch
    dev = on_device("d_x", d_x, dtypes=(torch.float32,))
    if d_x.dim() != 2:
        raise ValueError(f"d_x has shape {tuple(d_x.shape)}, expected (T, hidden)")
    T, H = d_x.shape
    bf = (torch.bfloat16,)
    on_device("d_gate", d_gate, dev, bf)
    if d_gate.dim() != 2 or d_gate.shape[1] != H:
        raise ValueError(f"d_gate has shape {tuple(d_gate.shape)}, expected (intermediate, {H})")
    I = d_gate.shape[0]
    on_device("d_up", d_up, dev, bf, (I, H))
    on_device("d_down", d_down, dev, bf)
    if d_down.dim() != 2 or d_down.shape[1] != I:
        raise ValueError(f"d_down has shape {tuple(d_down.shape)}, expected (out, {I})")
    O = d_down.shape[0]
    if d_residual is not None:
        on_device("d_residual", d_residual, dev, (torch.float32,), (T, O))
    with launch(dev, stream) as st:
        if d_out is None:
            d_out = torch.empty(T, O, dtype=torch.float32, device=dev)
        else:
            on_device("d_out", d_out, dev, (torch.float32,), (T, O))
        scratch = _scratch("objb_ffn_bf16_tokens_scratch_bytes", dev, d_gate.data_ptr(), d_up.data_ptr(),
                           d_down.data_ptr(), H, I, O, T)
        _lib.call("objb_ffn_bf16_tokens_device", d_gate.data_ptr(), d_up.data_ptr(), d_down.data_ptr(), H, I, O,
                  d_x.data_ptr(), T, _p(d_residual), d_out.data_ptr(), float(swiglu_limit), _p(scratch),
                  scratch.numel() if scratch is not None else 0, st)
    return d_out
