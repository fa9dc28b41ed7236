"""Refusals of the dense products and the router-training entry points: every
one is made on the host before anything is launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from objeta_b200 import CudaError, _lib, dense, router  # noqa: E402

P = 4096  # a non-null address that no refused call reads


def _fails(kind, text, name, *args):
    with pytest.raises(CudaError) as e:
        _lib.call(name, *args)
    assert e.value.kind == kind and text in e.value.source_message, e.value


def _linear(x=P, w=P, y=P, scratch=None, scratch_bytes=0, **f):
    d = dense._LinearDesc(tokens=4, in_features=64, out_features=32, x_dtype=2, w_dtype=2, y_dtype=2)
    for k, v in f.items():
        setattr(d, k, v)
    return ("objb_linear_device", ctypes.byref(d), x, w, f.get("bias"), None, y, None, scratch, scratch_bytes, None)


@pytest.mark.parametrize("kind,text,fields", [
    ("InvalidInput", "in_features", dict(in_features=0)),
    ("InvalidInput", "out_features", dict(out_features=(1 << 24) + 1)),
    ("InvalidInput", "tokens", dict(tokens=(1 << 30) + 1)),
    ("InvalidInput", "unknown activation 9", dict(activation=9)),
    ("InvalidInput", "unknown activation -1", dict(activation=-1)),
    ("InvalidInput", "reserved", dict(reserved=1)),
    ("Unsupported", "both bf16", dict(x_dtype=2, w_dtype=1)),
    ("Unsupported", "both bf16", dict(x_dtype=0, w_dtype=1)),
    ("Unsupported", "both bf16", dict(x_dtype=3, w_dtype=3)),
    ("Unsupported", "both bf16", dict(x_dtype=77, w_dtype=77)),
    ("Unsupported", "y is f32", dict(y_dtype=1)),
    ("Unsupported", "y is f32", dict(x_dtype=0, y_dtype=2)),
    ("InvalidInput", "x_stride", dict(x_stride=63)),
    ("InvalidInput", "w_stride", dict(w_stride=1)),
    ("InvalidInput", "y_stride", dict(y_stride=31)),
    ("InvalidInput", "null device pointer", dict(x=None)),
    ("InvalidInput", "null device pointer", dict(w=None)),
    ("InvalidInput", "null device pointer", dict(y=None)),
])
def test_linear_refusals(kind, text, fields):
    _fails(kind, text, *_linear(**fields))


def test_linear_null_descriptor_and_types():
    _fails("InvalidInput", "null descriptor", "objb_linear_device", None, P, P, None, None, P, None, None, 0, None)
    d = dense._LinearDesc(tokens=1, in_features=8, out_features=8, x_dtype=2, w_dtype=2, y_dtype=2, bias_dtype=1)
    _fails("Unsupported", "bias", "objb_linear_device", ctypes.byref(d), P, P, P, None, P, None, None, 0, None)
    d = dense._LinearDesc(tokens=1, in_features=8, out_features=8, x_dtype=2, w_dtype=2, y_dtype=2)
    _fails("InvalidInput", "same array", "objb_linear_device", ctypes.byref(d), P, P, None, None, P, P, None, 0, None)
    d.residual_stride = 9
    _fails("InvalidInput", "in place", "objb_linear_device", ctypes.byref(d), P, P, None, P, P, None, None, 0, None)
    _fails("InvalidInput", "null output", "objb_linear_scratch_bytes", ctypes.byref(d), P, P, None)


def _backward(**f):
    ptr = {k: f.pop(k, P) for k in ("dy", "z", "x", "w", "dx", "dw", "db")}
    d = dense._LinearBackwardDesc(tokens=4, in_features=64, out_features=32, x_dtype=2, w_dtype=2, dy_dtype=2,
                                  dw_dtype=2, outputs=7)
    for k, v in f.items():
        setattr(d, k, v)
    return ("objb_linear_backward_device", ctypes.byref(d), *ptr.values(), None, 0, None)


@pytest.mark.parametrize("kind,text,fields", [
    ("InvalidInput", "in_features", dict(in_features=0)),
    ("InvalidInput", "outputs", dict(outputs=0)),
    ("InvalidInput", "outputs", dict(outputs=8)),
    ("InvalidInput", "reserved", dict(reserved=3)),
    ("Unsupported", "dw is f32", dict(dw_dtype=1)),
    ("Unsupported", "dy is f32", dict(dy_dtype=1)),
    ("InvalidInput", "dx_stride", dict(dx_stride=3)),
    ("InvalidInput", "dw_stride", dict(dw_stride=3)),
    ("InvalidInput", "null device pointer", dict(dy=None)),
    ("InvalidInput", "null device pointer", dict(z=None, activation=2)),
    ("InvalidInput", "null device pointer", dict(x=None)),
    ("InvalidInput", "null device pointer", dict(dx=None)),
    ("InvalidInput", "null device pointer", dict(dw=None)),
    ("InvalidInput", "null device pointer", dict(db=None)),
])
def test_backward_refusals(kind, text, fields):
    _fails(kind, text, *_backward(**fields))


def test_ffn_refusals():
    _fails("InvalidInput", "in_features", "objb_ffn_bf16_tokens_device", P, P, P, 0, 8, 8, P, 1, None, P, 0.0, None, 0,
           None)
    _fails("InvalidInput", "null device pointer", "objb_ffn_bf16_tokens_device", P, None, P, 8, 8, 8, P, 1, None, P,
           0.0, None, 0, None)


def _bal(E=8, k=2, S=1, func=0, T=4, ld=0, off=None, logits=P):
    return ("objb_balance_loss_device", logits, ld, P, None, off, S, T, E, k, func, P, P, P, P, None, 0, None)


def _bwd(E=8, k=2, S=1, func=0, T=4, ld=0, ldo=0, off=None, dw=P, counts=None, scales=None, bg=0.0, zg=0.0, out=P + 64):
    return ("objb_router_backward_device", P, ld, P, dw, None, off, S, counts, scales, T, E, k, func, 0, 1.0, bg, zg,
            out, ldo, None)


@pytest.mark.parametrize("text,f", [
    ("top_k", dict(k=9)), ("top_k", dict(k=0)), ("num_experts", dict(E=0)), ("num_experts", dict(E=8193)),
    ("num_tokens", dict(T=(1 << 30) + 1)), ("score_func", dict(func=3)), ("score_func", dict(func=-1)),
    ("num_seqs", dict(S=0)), ("num_seqs", dict(S=2)), ("num_seqs", dict(S=(1 << 24) + 1, off=P)), ("num_seqs", dict(S=1 << 24, E=8192, off=P)),
])
def test_router_refusals(text, f):
    _fails("InvalidInput", text, *_bal(**f))
    _fails("InvalidInput", text, *_bwd(**f))


def test_router_more_refusals():
    _fails("InvalidInput", "logits_stride", *_bal(ld=7))
    _fails("InvalidInput", "null device pointer", *_bal(logits=None))
    _fails("InvalidInput", "row stride", *_bwd(ld=7))
    _fails("InvalidInput", "row stride", *_bwd(ldo=7))
    _fails("InvalidInput", "in place", *_bwd(out=P, ldo=12))
    _fails("InvalidInput", "come together", *_bwd(counts=P))
    _fails("InvalidInput", "needs the counts", *_bwd(bg=1.0))
    _fails("InvalidInput", "needs the counts", *_bwd(zg=1.0))
    _fails("InvalidInput", "neither", *_bwd(dw=None))
    _fails("InvalidInput", "top_k", "objb_moe_combine_backward_device", P, P, 4, P, 2, 0, 8, P, None)
    _fails("InvalidInput", "out_dim", "objb_moe_combine_backward_device", P, P, 4, P, 2, 2, 0, P, None)
    _fails("InvalidInput", "no value rows", "objb_moe_combine_backward_device", P, P, 0, P, 2, 2, 8, P, None)
    _fails("InvalidInput", "null", "objb_moe_combine_backward_device", P, None, 4, P, 2, 2, 8, P, None)


def test_python_refusals_without_a_gpu():
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dense.linear(x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dense.linear_backward(x, x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dense.ffn_bf16_tokens(x, x, x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        router.balance_loss(x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        router.router_backward(x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        router.moe_combine_backward(x, x, x)
    with pytest.raises(ValueError, match="unknown activation"):
        dense._activation("tanh")
