"""Dense products of many tokens: ``linear`` with bias, activation and residual
in its epilogue, its gradients, and the shared expert of a batch.

The reference's dense paths run one token (``gemv_bf16_device``,
``ffn_bf16_device``); these take T of them: the router's projection, the
shared expert beside ``moe_pairs``, an output head.  Types: x and w both bf16,
both f16, x f32 with w bf16, or both f32; y f32 or, where x is a 16-bit type,
that type.  Any sizes, row strides and element-aligned addresses.  Results
given by the caller overlap neither each other nor what the call reads, but
where it says so.  Results carry no autograd graph: a training loop calls
``linear_backward`` itself.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from ._launch import matrix, on_device, run

c_size = ctypes.c_size_t
c_int = ctypes.c_int
c_int32 = ctypes.c_int32
c_float = ctypes.c_float
c_void_p = ctypes.c_void_p

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_DX, _DW, _DBIAS = 1, 2, 4
# objb_linear_desc and objb_linear_backward_desc, field by field
_LINEAR = struct.Struct("@3N6i5N")
_BACKWARD = struct.Struct("@3N8i6N")


class _LinearDesc(ctypes.Structure):
    """objb_linear_desc (what _LINEAR packs)."""
    _fields_ = ([(n, c_size) for n in ("tokens", "in_features", "out_features")]
                + [(n, c_int32) for n in ("x_dtype", "w_dtype", "y_dtype", "bias_dtype", "activation", "reserved")]
                + [(n, c_size) for n in ("x_stride", "w_stride", "y_stride", "residual_stride", "z_stride")])


class _LinearBackwardDesc(ctypes.Structure):
    """objb_linear_backward_desc (what _BACKWARD packs)."""
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

_codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _dtype_code(name, dtype):
    code = _codes.get(dtype)
    if code is None:
        raise ValueError(f"{name} is {dtype}, expected torch.float32, torch.float16 or torch.bfloat16")
    return code


def _activation(name):
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"unknown activation {name!r}, expected one of {', '.join(ACTIVATIONS)}")
    return code


def _scratch(call, device, *args):
    n = c_size()
    _lib.call(call, *args, ctypes.byref(n))
    return torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None


def linear(d_x, d_w, d_bias=None, activation: str = "none", d_residual=None, out_dtype=None, d_y=None, d_z=None,
           stream=None):
    """y = act(d_x d_w^T + d_bias) + d_residual.

    d_x [T, in], d_w [out, in], d_bias [out] (f32 or d_w's type), d_residual
    [T, out] of y's type (may be ``d_y`` itself).  ``activation``: "none",
    "relu", "silu", "gelu" (erf) or "gelu_tanh".  ``out_dtype`` defaults to
    d_x's type.  ``d_z`` [T, out], of y's type, receives d_x d_w^T + d_bias for
    ``linear_backward``.
    """
    T, K, ldx = matrix("d_x", d_x)
    dev = d_x.device
    N, kw, ldw = matrix("d_w", d_w, dev)
    if kw != K:
        raise ValueError(f"d_w has shape {tuple(d_w.shape)}, expected (out, {K})")
    if d_y is not None and out_dtype is not None and d_y.dtype != out_dtype:
        raise ValueError(f"d_y is {d_y.dtype}, out_dtype {out_dtype}")
    head = (_dtype_code("d_x", d_x.dtype), _dtype_code("d_w", d_w.dtype))
    return run(dev, stream, _linear, T, K, N, ldx, ldw, head, _activation(activation), d_x, d_w, d_bias, d_residual,
               out_dtype or d_x.dtype, d_y, d_z, dev)


def _linear(st, T, K, N, ldx, ldw, head, act, d_x, d_w, d_bias, d_residual, ydt, d_y, d_z, dev):
    if d_y is None:
        d_y, ldy = torch.empty(T, N, dtype=ydt, device=dev), N
    else:
        ydt = d_y.dtype
        ldy = matrix("d_y", d_y, dev, None, (T, N))[2]
    bdt = ldr = ldz = 0
    bias = res = z = scratch = None
    if d_bias is not None:
        on_device("d_bias", d_bias, dev, shape=(N,))
        bdt, bias = _dtype_code("d_bias", d_bias.dtype), d_bias.data_ptr()
    if d_residual is not None:
        ldr = matrix("d_residual", d_residual, dev, (ydt,), (T, N))[2]
        res = d_residual.data_ptr()
    if d_z is not None:
        ldz = matrix("d_z", d_z, dev, (ydt,), (T, N))[2]
        z = d_z.data_ptr()
    x, w = d_x.data_ptr(), d_w.data_ptr()
    desc = _LINEAR.pack(T, K, N, *head, _dtype_code("d_y", ydt), bdt, act, 0, ldx, ldw, ldy, ldr, ldz)
    if head[0] == 0 or (x | w) & 15 or (ldx | ldw) & 7:  # an operand that has to be laid out again
        scratch = _scratch("objb_linear_scratch_bytes", dev, desc, x, w)
    _lib.call("objb_linear_device", desc, x, w, bias, res, d_y.data_ptr(), z,
              *((None, 0) if scratch is None else (scratch.data_ptr(), scratch.numel())), st)
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
    T, N, lddy = matrix("d_dy", d_dy)
    dev = d_dy.device
    nw, K, ldw = matrix("d_w", d_w, dev)
    if nw != N:
        raise ValueError(f"d_w has shape {tuple(d_w.shape)}, expected ({N}, in)")
    ldx = matrix("d_x", d_x, dev, None, (T, K))[2]
    act = _activation(activation)
    if act and d_z is None:
        raise ValueError(f"the gradient of {activation!r} needs d_z")
    if accumulate and ((need_dw and d_dw is None) or (need_dbias and d_dbias is None)):
        raise ValueError("accumulate needs the d_dw and d_dbias to add to")
    if need_dw and d_dw is not None and dw_dtype is not None and d_dw.dtype != dw_dtype:
        raise ValueError(f"d_dw is {d_dw.dtype}, dw_dtype {dw_dtype}")
    return run(dev, stream, _linear_backward, T, K, N, lddy, ldx, ldw, act, d_dy, d_x, d_w, d_z, need_dx, need_dw,
               need_dbias, dw_dtype or d_w.dtype, d_dx, d_dw, d_dbias, accumulate, dev)


def _linear_backward(st, T, K, N, lddy, ldx, ldw, act, d_dy, d_x, d_w, d_z, need_dx, need_dw, need_dbias, dw_dtype,
                     d_dx, d_dw, d_dbias, accumulate, dev):
    ldz = lddx = lddw = outputs = 0
    z = dx = dw = db = None
    wdt = gdt = _dtype_code("d_w", d_w.dtype)
    if act:
        ldz = matrix("d_z", d_z, dev, (d_dy.dtype,), (T, N))[2]
        z = d_z.data_ptr()
    if need_dx:
        if d_dx is None:
            d_dx, lddx = torch.empty(T, K, dtype=d_x.dtype, device=dev), K
        else:
            lddx = matrix("d_dx", d_dx, dev, (d_x.dtype,), (T, K))[2]
        dx, outputs = d_dx.data_ptr(), _DX
    if need_dw:
        if d_dw is None:
            d_dw, lddw = torch.empty(N, K, dtype=dw_dtype, device=dev), K
        else:
            lddw = matrix("d_dw", d_dw, dev, None, (N, K))[2]
        dw, outputs, gdt = d_dw.data_ptr(), outputs | _DW, _dtype_code("d_dw", d_dw.dtype)
    if need_dbias:
        if d_dbias is None:
            d_dbias = torch.empty(N, dtype=torch.float32, device=dev)
        else:
            on_device("d_dbias", d_dbias, dev, (torch.float32,), (N,))
        db, outputs = d_dbias.data_ptr(), outputs | _DBIAS
    desc = _BACKWARD.pack(T, K, N, _dtype_code("d_x", d_x.dtype), wdt, _dtype_code("d_dy", d_dy.dtype), gdt, act,
                          outputs, int(bool(accumulate)), 0, lddy, ldz, ldx, ldw, lddx, lddw)
    dy, x, w = d_dy.data_ptr(), d_x.data_ptr(), d_w.data_ptr()
    scratch = _scratch("objb_linear_backward_scratch_bytes", dev, desc, dy, x, w)
    _lib.call("objb_linear_backward_device", desc, dy, z, x, w, dx, dw, db,
              *((None, 0) if scratch is None else (scratch.data_ptr(), scratch.numel())), st)
    return d_dx if need_dx else None, d_dw if need_dw else None, d_dbias if need_dbias else None


_F32, _BF16 = (torch.float32,), (torch.bfloat16,)


def ffn_bf16_tokens(d_gate, d_up, d_down, d_x, d_residual=None, d_out=None, swiglu_limit: float = 0.0, stream=None):
    """``ffn_bf16_device`` for T tokens (the shared expert of a batch):
    out[t] = d_residual[t] + down SwiGLU(gate x_t, up x_t).

    d_gate, d_up [I, H] and d_down [O, I] bf16, d_x f32 [T, H], d_residual f32
    [T, O] or None; ``d_out`` may be ``d_residual`` or ``d_x`` itself.  f32 precision
    throughout, as the one-token call.  With ``swiglu_limit`` infinities are
    clamped and NaN stays NaN (the one-token call clamps it, as the reference).
    """
    dev = on_device("d_x", d_x, None, _F32)
    if d_x.dim() != 2:
        raise ValueError(f"d_x has shape {tuple(d_x.shape)}, expected (T, hidden)")
    T, H = d_x.shape
    on_device("d_gate", d_gate, dev, _BF16)
    if d_gate.dim() != 2 or d_gate.shape[1] != H:
        raise ValueError(f"d_gate has shape {tuple(d_gate.shape)}, expected (intermediate, {H})")
    I = d_gate.shape[0]
    on_device("d_up", d_up, dev, _BF16, (I, H))
    on_device("d_down", d_down, dev, _BF16)
    if d_down.dim() != 2 or d_down.shape[1] != I:
        raise ValueError(f"d_down has shape {tuple(d_down.shape)}, expected (out, {I})")
    return run(dev, stream, _ffn, T, H, I, d_down.shape[0], d_gate, d_up, d_down, d_x, d_residual, d_out,
               float(swiglu_limit), dev)


def _ffn(st, T, H, I, O, d_gate, d_up, d_down, d_x, d_residual, d_out, limit, dev):
    res = None
    if d_residual is not None:
        on_device("d_residual", d_residual, dev, _F32, (T, O))
        res = d_residual.data_ptr()
    if d_out is None:
        d_out = torch.empty(T, O, dtype=torch.float32, device=dev)
    else:
        on_device("d_out", d_out, dev, _F32, (T, O))
    g, u, d = d_gate.data_ptr(), d_up.data_ptr(), d_down.data_ptr()
    scratch = _scratch("objb_ffn_bf16_tokens_scratch_bytes", dev, g, u, d, H, I, O, T)
    _lib.call("objb_ffn_bf16_tokens_device", g, u, d, H, I, O, d_x.data_ptr(), T, res, d_out.data_ptr(), limit,
              *((None, 0) if scratch is None else (scratch.data_ptr(), scratch.numel())), st)
    return d_out
