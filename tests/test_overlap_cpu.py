"""Results over operands are refused on the host; arrays that only lie near one another are not."""
import ctypes
import itertools

import pytest

torch = pytest.importorskip("torch")

from objeta_b200 import CudaError, _lib, dense, router  # noqa: E402,F401

M = 1 << 20  # addresses that no refused call reads


def _status(name, *args):
    """The refusal's text; the calls below that are not refused for an overlap have a scratch too small (or, of
    the router's, no device) to go on to a launch."""
    with pytest.raises(CudaError) as e:
        _lib.call(name, *args)
    return e.value.source_message


def _linear(x=M, w=2 * M, bias=None, res=None, y=3 * M, z=None, **f):
    d = dense._LinearDesc(tokens=4, in_features=60, out_features=60, x_dtype=2, w_dtype=2, y_dtype=2, bias_dtype=2)
    for k, v in f.items():
        setattr(d, k, v)
    return _status("objb_linear_device", ctypes.byref(d), x, w, bias, res, y, z, 256, 1, None)


ROW = 60 * 2


@pytest.mark.parametrize("args", [
    dict(y=M), dict(y=M + ROW), dict(y=M + 3 * ROW + ROW - 2), dict(y=M - 2 * ROW), dict(y=2 * M + 59 * ROW),
    dict(bias=3 * M + 4), dict(z=3 * M + 2 * ROW), dict(z=M), dict(z=2 * M), dict(res=3 * M + ROW), dict(res=4 * M, z=4 * M),
    dict(x_stride=200, y_stride=200, y=M + ROW - 2), dict(x_stride=200, y_stride=200, y=M + 400 - 2),
    dict(x_stride=200, y_stride=200, y=M - 400 + 400 - ROW + 2), dict(x_stride=200, y=M + ROW), dict(x_stride=64, y=M + 130),
])
def test_linear_overlaps(args):
    assert "overlaps" in _linear(**args)


@pytest.mark.parametrize("args", [
    dict(), dict(y=M + 4 * ROW), dict(y=M - 4 * ROW), dict(bias=4 * M, z=5 * M, res=3 * M), dict(res=M), dict(res=2 * M),
    dict(x_stride=200, y_stride=200, y=M + ROW), dict(x_stride=200, y_stride=200, y=M + 400 - ROW),
    dict(x_stride=200, y_stride=200, y=M - 400 + ROW), dict(x_stride=400, y=M + ROW), dict(x_stride=400, w=M + ROW, y_stride=61),
    dict(x_stride=300, y_stride=302, y=M + ROW),  # among one another with different strides: not looked through
])
def test_linear_neighbours(args):
    assert "overlaps" not in _linear(**args)


def _bytes(p, rows, width, pitch):
    return {p + r * pitch + i for r in range(rows) for i in range(width)}


def test_linear_against_every_byte():
    """Small arrays at every offset, against the sets of their bytes (equal strides, and contiguous ones)."""
    for ldx, ldy in ((3, 3), (7, 7), (4, 4), (7, 3), (3, 7), (9, 3), (3, 9)):
        for tx, off in itertools.product((1, 3), range(-60, 61, 2)):
            d = dense._LinearDesc(tokens=tx, in_features=3, out_features=3, x_dtype=2, w_dtype=2, y_dtype=2,
                                  x_stride=ldx, y_stride=ldy)
            msg = _status("objb_linear_device", ctypes.byref(d), M, 2 * M, None, None, M + off, None, 256, 1, None)
            share = bool(_bytes(M, tx, 6, 2 * ldx) & _bytes(M + off, tx, 6, 2 * ldy))
            assert ("overlaps" in msg) == share, (ldx, ldy, tx, off)


def _backward(outputs=7, act=0, dy=M, z=2 * M, x=3 * M, w=4 * M, dx=5 * M, dw=6 * M, db=7 * M):
    d = dense._LinearBackwardDesc(tokens=300, in_features=60, out_features=60, x_dtype=2, w_dtype=2, dy_dtype=2,
                                  dw_dtype=2, outputs=outputs, activation=act)
    return _status("objb_linear_backward_device", ctypes.byref(d), dy, z, x, w, dx, dw, db, 256, 1, None)


@pytest.mark.parametrize("args", [dict(dx=M), dict(dw=M + 8), dict(db=M), dict(dx=3 * M), dict(dw=4 * M), dict(dw=3 * M),
                                  dict(dx=4 * M), dict(act=2, dx=2 * M), dict(dx=6 * M), dict(db=6 * M + 4),
                                  dict(outputs=1, dx=4 * M), dict(outputs=2, dw=3 * M)])
def test_backward_overlaps(args):
    assert "overlaps" in _backward(**args)


@pytest.mark.parametrize("args", [dict(), dict(dx=2 * M), dict(outputs=1, dx=3 * M, dw=M), dict(outputs=2, dw=4 * M, dx=M)])
def test_backward_neighbours(args):
    """What a call does not read may be written: z without an activation, x without dw, w without dx."""
    assert "overlaps" not in _backward(**args)


def test_ffn():
    def ffn(x=M, res=None, out=5 * M):
        return _status("objb_ffn_bf16_tokens_device", 2 * M, 3 * M, 4 * M, 64, 32, 64, x, 300, res, out, 0.0, 256, 1, None)
    for bad in (dict(out=2 * M), dict(out=3 * M + 64), dict(out=4 * M), dict(out=5 * M, res=5 * M + 4)):
        assert "overlaps" in ffn(**bad)
    for good in (dict(), dict(out=M), dict(res=5 * M), dict(out=M, res=M)):
        assert "overlaps" not in ffn(**good)


def test_router():
    def bwd(logits=M, ids=2 * M, dw=3 * M, mask=None, off=None, counts=None, scales=None, out=4 * M, ldo=0):
        return ("objb_router_backward_device", logits, ldo, ids, dw, mask, off, 1, counts, scales, 4, 8, 2, 0, 0, 1.0, 0.0,
                0.0, out, ldo, None)
    for bad in (dict(out=M + 4), dict(out=2 * M), dict(out=3 * M + 8), dict(out=M + 8 * 4, ldo=12), dict(mask=4 * M + 1),
                dict(off=4 * M), dict(counts=4 * M, scales=5 * M), dict(counts=5 * M, scales=4 * M)):
        assert "overlaps" in _status(*bwd(**bad)), bad
    args = ("objb_moe_combine_backward_device", M, 2 * M, 4, 3 * M, 4, 2, 8)
    for bad in (M, 2 * M + 4, 3 * M):
        assert "overlaps" in _status(*args, bad, None)
